"""Bounded-cache operators on the CPU: the line of tiles, the plain forms, and every refusal before a launch."""

import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import flashdec_amd as fd
from flashdec_amd import _lib, bounded
from oracle.attention import paged_decode_attention as oracle_decode
from tests import bounded_oracle as ob
from tests.helpers import make_paged_inputs, np32

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_a_rows_line_holds_each_attended_tile_once(tmp_path):
    exe = tmp_path / "bounded_row_host"
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", str(ROOT / "flashdec_amd" / "csrc"),
                    str(ROOT / "tests" / "native" / "bounded_row_host.cpp"), "-o", str(exe)], check=True)
    ran = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert ran.returncode == 0, ran.stderr


def test_plain_forms_agree_with_the_decode_oracle_and_each_other():
    q, k, v, table, lens = make_paged_inputs([70, 0, 33], 4, 2, 64, 16, device="cpu", seed=2)
    want = oracle_decode(np32(q), np32(k), np32(v), table.numpy(), lens.numpy())
    out, weights = ob.attend(q, k, v, table, lens)
    assert torch.allclose(out, torch.from_numpy(want).double(), atol=1e-5)
    assert torch.allclose(weights.sum(dim=2), torch.tensor([[2.0, 2.0], [0.0, 0.0], [2.0, 2.0]]).double())
    wide, _ = ob.attend(q, k, v, table, lens, window=1000, sinks=3)
    assert torch.equal(wide, out)
    # eviction, then attention over what is left, is attention over the kept tokens
    kept, new_lens, _, k2, v2 = ob.evict(k, v, table, lens, torch.rand(3, 2, 80), 20, 4, 6)
    cut, _ = ob.attend(q, k2, v2, table, new_lens)
    for b, h in ((0, 0), (0, 1), (2, 1)):
        at = kept[b, h].long()
        keys, values = (c[table[b, at // 16].long(), h, at % 16].double() for c in (k, v))
        p = torch.softmax(q[b, 2 * h:2 * h + 2].double() @ keys.t() / 8.0, dim=1)
        assert torch.allclose(cut[b, 2 * h:2 * h + 2], p @ values)


def test_kept_tokens_order():
    nan, inf = math.nan, math.inf
    score = [9.0, nan, -inf, 0.0, -0.0, 1.0, 1.0, inf, 0.5, nan]
    assert ob.kept_tokens(score, 10, 3, 0, 0) == [0, 5, 7]  # the first of the two ones
    assert ob.kept_tokens(score, 10, 6, 0, 0) == [0, 3, 5, 6, 7, 8]  # the lower of the equal zeros
    assert ob.kept_tokens(score, 10, 9, 0, 0) == [0, 1, 2, 3, 4, 5, 6, 7, 8]  # NaN behind -inf, the lower first
    assert ob.kept_tokens(score, 10, 4, 2, 2) == [0, 1, 8, 9]
    assert ob.kept_tokens(score, 3, 4, 2, 2) == [0, 1, 2]


def test_cpu_tensors_are_refused():
    q, k, v, table, lens = make_paged_inputs([40, 8], 4, 2, 64, 16, device="cpu")
    scores = torch.zeros(2, 2, 48)
    with pytest.raises(ValueError, match="must be CUDA tensors"):
        fd.paged_decode_attention_window(q, k, v, table, lens, 8)
    with pytest.raises(ValueError, match="must be CUDA tensors"):
        fd.paged_decode_attention_scored(q, k, v, table, lens, scores)
    with pytest.raises(ValueError, match="must be CUDA tensors"):
        fd.paged_kv_evict(k, v, table, lens, scores, 16)


def test_arguments_that_are_no_tensors_are_refused():
    q, k, v, table, lens = make_paged_inputs([40, 8], 4, 2, 64, 16, device="cpu")
    with pytest.raises(TypeError, match="scores must be a torch.Tensor"):
        fd.paged_decode_attention_scored(q, k, v, table, lens, [[0.0]])
    for bad in (None, 3, [[0.0] * 48]):
        with pytest.raises(TypeError, match="must be torch.Tensors"):
            fd.paged_kv_evict(k, v, table, lens, bad, 16)
        with pytest.raises(TypeError, match="must be torch.Tensors"):
            fd.paged_kv_evict_into(k, v, table, lens, torch.zeros(2, 2, 48), 16, bad, torch.empty_like(lens))


def test_names_are_exported():
    for name in ("window", "window_into", "scored", "scored_into"):
        assert f"paged_decode_attention_{name}" in fd.__all__
        assert getattr(fd, f"paged_decode_attention_{name}") is getattr(bounded, f"paged_decode_attention_{name}")
    assert fd.paged_kv_evict is bounded.paged_kv_evict and fd.paged_kv_evict_into is bounded.paged_kv_evict_into


def test_score_table_checks():
    cpu = torch.device("cpu")
    good = torch.zeros(2, 3, 64)

    def check(t):
        bounded._check_scores(t, "scores", 2, 3, 64, cpu)

    check(good)
    check(torch.zeros(3, 2, 70).transpose(0, 1))  # any order of rows, more tokens than the tables
    check(torch.zeros(2, 3, 200)[:, :, 5:100])
    for bad, message in ((torch.zeros(2, 64), "shape"), (torch.zeros(1, 3, 64), "shape"), (torch.zeros(2, 2, 64), "shape"),
                         (torch.zeros(2, 3, 63), "every token"), (good.double(), "float32"), (good.half(), "float32"),
                         (torch.zeros(2, 64, 3).transpose(1, 2), "unit token stride"),
                         (torch.zeros(1, 3, 64).expand(2, 3, 64), "overlapping"),
                         (torch.zeros(2, 1, 64).expand(2, 3, 64), "overlapping")):
        with pytest.raises(ValueError, match=message):
            check(bad)
    with pytest.raises(ValueError, match="device"):
        bounded._check_scores(good, "scores", 2, 3, 64, torch.device("meta"))


def test_whole_numbers():
    assert bounded._whole(4, "window", 1) == 4
    for bad in (0, -1, True, 2.0, "8", None):
        with pytest.raises(ValueError, match="window must be an integer of at least 1"):
            bounded._whole(bad, "window", 1)


def test_overlaps_are_seen():
    t = torch.zeros(4, 6)
    assert bounded._spread_out(t) and bounded._spread_out(t.t()) and bounded._spread_out(t[::2, ::3])
    assert bounded._spread_out(torch.zeros(3, 0)) and bounded._spread_out(torch.zeros(1).expand(1, 1))
    assert not bounded._spread_out(t[:1].expand(4, 6)) and not bounded._spread_out(torch.zeros(9).as_strided((4, 3), (2, 1)))
    assert bounded._reach(t) == 96 and bounded._reach(t.t()) == 96 and bounded._reach(t[1:3, 2:4]) == 32


class _OnGpu(torch.Tensor):
    """A CPU tensor that passes for one on the GPU."""

    is_cuda = property(lambda self: True)


@pytest.fixture
def launches(monkeypatch):
    """Public calls on CPU tensors, up to their launch: (what was launched, as (entry's name, stream, workspace's
    address), a function that sets the current stream)."""
    ran, stream = [], [0]

    def run_on(handle):
        stream[0] = handle

    def launch(device, entry, *args):
        if entry in (_lib.paged_decode_window_floats, _lib.paged_decode_scored_floats):
            return entry(*args)
        *_, workspace, words, on = args
        ran.append((entry.__name__, on, workspace))

    monkeypatch.setattr(bounded, "_validate_inputs", lambda *args: None)
    monkeypatch.setattr(bounded, "_launch", launch)
    monkeypatch.setattr(bounded, "_capturing", lambda on: False)
    monkeypatch.setattr(bounded, "_WORKSPACES", type(bounded._WORKSPACES)())
    monkeypatch.setattr(bounded, "_LAST", type(bounded._LAST)())
    monkeypatch.setattr(_lib, "current_stream_handle", lambda device: stream[0])
    return ran, run_on


@pytest.mark.parametrize("op", ["window", "scored", "evict"])
def test_streams_share_no_workspace(launches, op):
    """The same call on several streams in turn: each stream's launches get a workspace that no other's get."""
    ran, run_on = launches
    q, k, v, table, lens = (t.as_subclass(_OnGpu) for t in make_paged_inputs([3000, 40], 16, 2, 128, 32, device="cpu"))
    scores = torch.zeros(2, 2, table.shape[1] * 32).as_subclass(_OnGpu)
    kept, new = torch.empty(2, 2, 64, dtype=torch.int32), torch.empty_like(lens)

    def call():
        if op == "window":
            fd.paged_decode_attention_window(q, k, v, table, lens, 2000, 4)
        elif op == "scored":
            fd.paged_decode_attention_scored(q, k, v, table, lens, scores)
        else:
            fd.paged_kv_evict_into(k, v, table, lens, scores, 64, kept, new, 4, 16)

    for _ in range(3):
        for on in (0, 1 << 12, 1 << 13):
            run_on(on)
            call()
    assert [on for _, on, _ in ran] == 3 * [0, 1 << 12, 1 << 13]
    assert all(workspace for _, _, workspace in ran)
    assert len({workspace for _, _, workspace in ran[:3]}) == 3
    assert ran[3:6] == ran[:3] and ran[6:] == ran[:3]


# ----------------------------------------------------------------- C entry points --
def _decode_args(**over):
    a = _lib.PagedDecodeArgs()
    a.struct_size = ctypes.sizeof(a)
    a.dtype = _lib.FD_DTYPE_BF16
    a.num_seqs, a.num_q_heads, a.num_kv_heads, a.head_dim = 2, 16, 2, 128
    a.block_size, a.num_blocks, a.max_blocks_per_seq = 32, 100, 64
    a.q = a.k_cache = a.v_cache = a.block_tables = a.seq_lens = a.out = 0x10000
    a.num_splits = 1
    for name, value in over.items():
        setattr(a, name, value)
    return a


def _window(window=1500, sinks=4, size=None):
    return _lib.WindowArgs(struct_size=ctypes.sizeof(_lib.WindowArgs) if size is None else size, window=window,
                           sink_tokens=sinks)


def _scores(tokens=2048, scores=0x10000, size=None):
    return _lib.ScoreArgs(struct_size=ctypes.sizeof(_lib.ScoreArgs) if size is None else size, scores=scores,
                          stride=(4096, 2048), tokens=tokens)


def _refused(rc, lib, text, code=-1):
    assert rc == code, (rc, lib.fd_last_error())
    assert text in lib.fd_last_error().decode(), lib.fd_last_error()


def test_window_entry_refusals():
    lib = _lib.load_library()
    a, floats = _decode_args(), ctypes.c_int64()
    ref = ctypes.byref
    assert lib.fd_paged_decode_window_floats(ref(a), ref(_window()), ref(floats)) == 0 and floats.value > 0
    need = floats.value
    call = lib.fd_paged_decode_window
    _refused(call(None, ref(_window()), 16, need, None), lib, "args is NULL")
    _refused(call(ref(a), None, 16, need, None), lib, "window is NULL")
    _refused(call(ref(a), ref(_window(size=3)), 16, need, None), lib, "struct_size")
    for window, sinks in ((0, 0), (-5, 0), (5, -1)):
        _refused(call(ref(a), ref(_window(window, sinks)), 16, need, None), lib, "window must be positive")
    for ws, n in ((None, need), (16, need - 1), (24, need)):
        _refused(call(ref(a), ref(_window()), ws, n, None), lib, "workspace")
    _refused(lib.fd_paged_decode_window_floats(ref(a), ref(_window()), None), lib, "floats is NULL")
    for over, text, code in (({"num_splits": 2}, "split", -1), ({"balance_target": 4}, "balance_target", -1),
                             ({"split_counters": 0x100}, "counters", -1), ({"head_dim": 96}, "head_dim", -2),
                             ({"block_size": 64}, "block_size", -2), ({"num_kv_heads": 3}, "divisible", -1),
                             ({"max_blocks_per_seq": 1 << 27}, "2^31", -2), ({"dtype": 2}, "dtype", -2),
                             ({"append_k": 64, "append_v": 64, "slot_mapping": 64}, "append", -2),
                             ({"kv_reuse": 2}, "kv_reuse", -1)):
        _refused(call(ref(_decode_args(**over)), ref(_window()), 16, need, None), lib, text, code)


def test_windows_and_sinks_without_an_end():
    """Any window and sink count past the longest row, up to the largest number, plans as 2^31 - 1 does."""
    lib, ref, floats = _lib.load_library(), ctypes.byref, ctypes.c_int64()

    def need(a, window, sinks):
        floats.value = -1
        assert lib.fd_paged_decode_window_floats(ref(a), ref(_window(window, sinks)), ref(floats)) == 0
        return floats.value

    huge = (2**31, 2**32, 2**62, 2**63 - 62, 2**63 - 1)
    for a in (_decode_args(), _decode_args(max_blocks_per_seq=(2**31 >> 5) - 200), _decode_args(num_q_heads=600)):
        all_of_it = need(a, 2**31 - 1, 0)
        assert all_of_it > 0
        for n in huge:
            for window, sinks in ((n, 0), (n, 4), (5, n), (n, n), (n, 2**31 - 1)):
                assert need(a, window, sinks) == all_of_it
                # and the launch asks for as much
                _refused(lib.fd_paged_decode_window(ref(a), ref(_window(window, sinks)), 16, all_of_it - 1, None), lib,
                         "workspace")


def test_scored_entry_refusals():
    lib = _lib.load_library()
    a, floats, ref = _decode_args(), ctypes.c_int64(), ctypes.byref
    assert lib.fd_paged_decode_scored_floats(ref(a), ref(floats)) == 0
    need = floats.value
    assert need >= 2 * 16 * 2048  # one float per query head and token at least
    call = lib.fd_paged_decode_scored
    _refused(call(ref(a), None, 16, need, None), lib, "scores is NULL")
    _refused(call(ref(a), ref(_scores(size=4)), 16, need, None), lib, "struct_size")
    _refused(call(ref(a), ref(_scores(scores=None)), 16, need, None), lib, "NULL tensor")
    _refused(call(ref(a), ref(_scores(tokens=2047)), 16, need, None), lib, "every token")
    for bad in (2, -1):
        table = _scores()
        table.ragged = bad
        _refused(call(ref(a), ref(table), 16, need, None), lib, "ragged must be 0 or 1")
    _refused(call(ref(a), ref(_scores()), 16, need - 1, None), lib, "workspace")
    _refused(call(ref(_decode_args(num_splits=3)), ref(_scores()), 16, need, None), lib, "split")
    _refused(lib.fd_paged_decode_scored_floats(None, ref(floats)), lib, "args is NULL")


def test_evict_entry_refusals():
    lib, ref = _lib.load_library(), ctypes.byref

    def args(**over):
        a = _lib.KvEvictArgs()
        a.struct_size = ctypes.sizeof(a)
        a.dtype = _lib.FD_DTYPE_BF16
        a.num_seqs, a.num_kv_heads, a.head_dim, a.block_size, a.num_blocks, a.max_blocks_per_seq = 2, 2, 128, 32, 9, 4
        for name in ("k_cache", "v_cache", "block_tables", "seq_lens", "scores", "kept", "new_scores"):
            setattr(a, name, 0x10000)
        a.new_seq_lens = 0x20000
        a.score_tokens, a.keep, a.sink_tokens, a.recent_tokens = 128, 64, 4, 16
        for name, value in over.items():
            setattr(a, name, value)
        return a

    words = ctypes.c_int64()
    assert lib.fd_kv_evict_words(ref(args()), ref(words)) == 0 and words.value > 0
    _refused(lib.fd_kv_evict_words(ref(args()), None), lib, "words is NULL")
    _refused(lib.fd_kv_evict(None, 16, words, None), lib, "args is NULL")
    for ws, n in ((None, words.value), (16, words.value - 1), (18, words.value)):
        _refused(lib.fd_kv_evict(ref(args()), ws, n, None), lib, "workspace")
    for over, text, code in (({"struct_size": 8}, "struct_size", -1), ({"dtype": 2}, "dtype", -2),
                             ({"num_seqs": 0}, "positive", -1), ({"head_dim": 80}, "head_dim", -2),
                             ({"block_size": 4}, "block_size", -2), ({"kept": None}, "NULL tensor", -1),
                             ({"new_scores": None}, "NULL tensor", -1), ({"keep": 0}, "keep", -1),
                             ({"keep": 19}, "keep", -1), ({"sink_tokens": -1}, "keep", -1),
                             ({"recent_tokens": -1}, "keep", -1), ({"score_tokens": 127}, "every token", -1),
                             ({"max_blocks_per_seq": 1 << 26, "score_tokens": 1 << 40}, "2^31", -2),
                             ({"max_blocks_per_seq": (1 << 26) - 1000, "score_tokens": 1 << 40}, "2^31", -2),
                             ({"keep": 1 << 31}, "2^31", -2), ({"new_seq_lens": 0x10000}, "must not be seq_lens", -1),
                             ({"num_seqs": 1 << 30}, "grid", -1)):
        _refused(lib.fd_kv_evict(ref(args(**over)), 16, 1 << 40, None), lib, text, code)


def _evict_args(**over):
    a = _lib.KvEvictArgs()
    a.struct_size = ctypes.sizeof(a)
    a.dtype = _lib.FD_DTYPE_BF16
    a.num_seqs, a.num_kv_heads, a.head_dim, a.block_size, a.num_blocks, a.max_blocks_per_seq = 2, 2, 128, 32, 9, 4
    for name in ("k_cache", "v_cache", "block_tables", "seq_lens", "scores", "kept", "new_scores"):
        setattr(a, name, 0x10000)
    a.new_seq_lens = 0x20000
    a.score_tokens, a.keep, a.sink_tokens, a.recent_tokens = 128, 64, 4, 16
    for name, value in over.items():
        setattr(a, name, value)
    return a


def test_sinks_and_recent_tokens_whose_sum_wraps():
    lib, words = _lib.load_library(), ctypes.c_int64()
    for sinks, recent in ((2**62, 2**62), (2**63 - 1, 2), (2, 2**63 - 1), (2**63 - 1, 2**63 - 1), (65, 0), (0, 65), (33, 32)):
        a = _evict_args(sink_tokens=sinks, recent_tokens=recent)
        _refused(lib.fd_kv_evict_words(ctypes.byref(a), ctypes.byref(words)), lib, "keep must be positive and hold")
        _refused(lib.fd_kv_evict(ctypes.byref(a), 16, 1 << 40, None), lib, "keep must be positive and hold")
    for sinks, recent in ((64, 0), (0, 64), (32, 32)):
        a = _evict_args(sink_tokens=sinks, recent_tokens=recent)
        assert lib.fd_kv_evict_words(ctypes.byref(a), ctypes.byref(words)) == 0 and words.value > 0


@pytest.mark.parametrize("over", [
    {"max_blocks_per_seq": 2**60}, {"max_blocks_per_seq": 2**59}, {"max_blocks_per_seq": 2**59 + 4},
    {"max_blocks_per_seq": 2**63 - 1}, {"num_seqs": 2**32, "num_kv_heads": 2**32}, {"num_seqs": 2**62, "num_kv_heads": 4},
    {"num_seqs": 2**63 - 1}])
def test_sizes_whose_products_wrap(over):
    """Refused by name; no division by a size that wrapped to zero."""
    lib, ref, n = _lib.load_library(), ctypes.byref, ctypes.c_int64()
    if "num_kv_heads" in over:
        over = {**over, "num_q_heads": over["num_kv_heads"]}
    what, code = ("2^31", -2) if "max_blocks_per_seq" in over else ("grid too large", -1)
    a = _decode_args(**over)
    _refused(lib.fd_paged_decode_window_floats(ref(a), ref(_window()), ref(n)), lib, what, code)
    _refused(lib.fd_paged_decode_scored_floats(ref(a), ref(n)), lib, what, code)
    _refused(lib.fd_paged_decode_window(ref(a), ref(_window()), 16, 1 << 62, None), lib, what, code)
    _refused(lib.fd_paged_decode_scored(ref(a), ref(_scores(2**63 - 1)), 16, 1 << 62, None), lib, what, code)
    over.pop("num_q_heads", None)
    a = _evict_args(score_tokens=2**63 - 1, **over)
    _refused(lib.fd_kv_evict_words(ref(a), ref(n)), lib, what, code)
    _refused(lib.fd_kv_evict(ref(a), 16, 1 << 62, None), lib, what, code)


def test_evictions_past_a_launch_dimension():
    """A launch dimension holds 2^32 - 1 threads: refused before the first kernel, which writes lengths and lists."""
    lib, ref = _lib.load_library(), ctypes.byref
    long = {"num_seqs": 1024, "num_kv_heads": 8, "max_blocks_per_seq": 1 << 13, "score_tokens": 1 << 18, "keep": 1 << 17}
    rows = {name: (1 << 22, 1 << 19, 128, 1) for name in ("k_stride", "v_stride")}
    dims = {name: (1 << 22, 1 << 19, 1, 32) for name in ("k_stride", "v_stride")}
    for over in ({**long, **rows}, {**long, **dims}, {"num_seqs": 1 << 22, "num_kv_heads": 1, **rows},
                 {"num_seqs": 1 << 21, "num_kv_heads": 2}):
        a = _evict_args(**{**over, **{name: (ctypes.c_int64 * 4)(*over[name]) for name in over if name.endswith("stride")}})
        _refused(lib.fd_kv_evict(ref(a), 16, 1 << 40, None), lib, "grid too large")


def test_decode_grids_past_a_launch_dimension():
    """The weights' launch of 2^24 short rows, and the rows of the element-by-element kernel."""
    lib, ref = _lib.load_library(), ctypes.byref
    heads = {"num_q_heads": 1, "num_kv_heads": 1, "block_size": 8, "max_blocks_per_seq": 1}
    a = _decode_args(num_seqs=1 << 24, **heads)
    _refused(lib.fd_paged_decode_scored(ref(a), ref(_scores(8)), 16, 1 << 40, None), lib, "grid too large", -2)
    a = _decode_args(num_seqs=1 << 26, **heads)
    _refused(lib.fd_paged_decode_window(ref(a), ref(_window()), 16, 1 << 40, None), lib, "grid too large", -2)


def test_more_heads_than_a_grid_dimension_holds():
    lib, ref, n = _lib.load_library(), ctypes.byref, ctypes.c_int64()
    for heads, taken in ((8 * 65535, True), (8 * 65535 + 1, False), (1 << 20, False), (2**31 - 1, False)):
        a = _decode_args(num_seqs=1, num_q_heads=heads, num_kv_heads=1)
        if taken:
            assert lib.fd_paged_decode_window_floats(ref(a), ref(_window()), ref(n)) == 0
            assert lib.fd_paged_decode_scored_floats(ref(a), ref(n)) == 0 and n.value > 0
            continue
        _refused(lib.fd_paged_decode_window_floats(ref(a), ref(_window()), ref(n)), lib, "grid too large", -2)
        _refused(lib.fd_paged_decode_scored_floats(ref(a), ref(n)), lib, "grid too large", -2)
        _refused(lib.fd_paged_decode_window(ref(a), ref(_window()), 16, 1 << 50, None), lib, "grid too large", -2)
        _refused(lib.fd_paged_decode_scored(ref(a), ref(_scores()), 16, 1 << 50, None), lib, "grid too large", -2)


LAYOUT_PROBE = r"""
#include <stddef.h>
#include <stdio.h>
#include "flashdec_hip.h"
#define F(S, f) printf(#S " " #f " %zu\n", offsetof(S, f));
int main(void) {
%s
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_argument_structs_match_c_layout(tmp_path):
    pairs = [("fd_window_args", _lib.WindowArgs), ("fd_score_args", _lib.ScoreArgs),
             ("fd_kv_evict_args", _lib.KvEvictArgs)]
    lines = [f"  F({c}, {name})" for c, py in pairs for name, _ in py._fields_]
    lines += [f'  printf("{c} sizeof %zu\\n", sizeof({c}));' for c, _ in pairs]
    src = tmp_path / "probe.c"
    src.write_text(LAYOUT_PROBE.replace("%s", "\n".join(lines)))
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", str(ROOT / "include"), str(src), "-o", str(exe)],
                   check=True)
    layout = {}
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        struct, field, value = line.split()
        layout[(struct, field)] = int(value)
    for c, py in pairs:
        assert layout[(c, "sizeof")] == ctypes.sizeof(py), c
        for name, _ in py._fields_:
            assert layout[(c, name)] == getattr(py, name).offset, (c, name)
