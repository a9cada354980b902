"""Block selection on the CPU: the score's two forms, the plain forms, and every refusal before a launch."""

import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import flashdec_amd as fd
from flashdec_amd import _lib, sparse
from tests import sparse_oracle as so
from tests.helpers import make_paged_inputs

HEADER = Path(__file__).resolve().parents[1] / "include" / "flashdec_hip.h"


def test_the_score_bounds_every_keys_and_its_two_forms_agree():
    q, k, _, table, lens = make_paged_inputs([160], 6, 2, 64, 16, device="cpu", seed=5)
    bounds = so.key_bounds(k, table, lens, torch.zeros(k.shape[0], 2, 2, 64, dtype=k.dtype))
    ids = table[0].tolist()
    for h in range(2):
        queries = q[0, 3 * h : 3 * h + 3].double()
        low, high = bounds[ids, h].double().unbind(1)
        plain = sum(torch.maximum(x * low, x * high).sum(dim=1) for x in queries)
        score = so.scores(queries, bounds[:, h], ids)
        assert torch.equal(score, plain.float())
        products = (k[ids, h].double() @ queries.t()).sum(dim=2)  # [block, token]
        assert bool((score.double() * (1 + 2.0**-23) + 2.0**-20 >= products.amax(dim=1)).all())


def test_plain_selection():
    bounds = torch.zeros(9, 1, 2, 64)
    bounds[:, 0, 1, 0] = torch.tensor([0.0, 5.0, 1.0, 1.0, 9.0, math.nan, 2.0, 0.0, 0.0])
    q = torch.zeros(1, 2, 64)
    q[0, :, 0] = 1.0
    table, lens = torch.arange(9)[None], torch.tensor([65])

    def chosen(n, sinks=0, recent=1, table=table, lens=lens):
        return so.select(q, bounds, table, lens, 8, n, sinks, recent, 1)

    assert chosen(3)[0][0, 0].tolist() == [4, 5, 8]
    assert chosen(6)[0][0, 0].tolist() == [1, 2, 4, 5, 6, 8]  # of the two ones the lower block
    assert chosen(5, 2, 2)[0][0, 0].tolist() == [0, 1, 5, 7, 8]
    assert chosen(9)[0][0, 0].tolist() == list(range(9)) and chosen(9)[2].item() == 65
    blocks, tables, n = chosen(4, table=torch.tensor([[0, 1, 2, 3, 99, 5, 6, 7, -1]]))
    assert blocks[0, 0].tolist() == [1, 5, 6, 8] and tables[0, 0].tolist() == [1, 5, 6, -1] and n.item() == 25


def test_the_step_between_a_pools_blocks():
    pool = torch.zeros(5, 3, 16, 64)
    assert sparse._block_step(pool) == 3 and sparse._block_step(pool[:, :1]) == 1
    assert sparse._block_step(torch.zeros(5, 2, 3, 16, 64)[:, 1]) == 6
    assert sparse._block_step(torch.zeros(5, 16, 3, 64).transpose(1, 2)) == 48
    for bad in (pool.transpose(0, 1), torch.zeros(5, 1, 16, 64).expand(5, 3, 16, 64),
                torch.zeros(5 * 3 * 16 * 64 + 999).as_strided((5, 3, 16, 64), (3100, 1024, 64, 1))):
        with pytest.raises(ValueError, match="block stride"):
            sparse._block_step(bad)
    view = sparse._one_head_blocks(pool, 3)
    pool.normal_()
    assert view.shape == (15, 1, 16, 64) and torch.equal(view[3 * 4 + 2, 0], pool[4, 2])


def test_cpu_tensors_and_arguments_that_are_no_tensors_are_refused():
    q, k, v, table, lens = make_paged_inputs([40, 8], 4, 2, 64, 16, device="cpu")
    bounds = torch.zeros(k.shape[0], 2, 2, 64, dtype=k.dtype)
    with pytest.raises(ValueError, match="must be CUDA tensors"):
        fd.paged_key_bounds(k, table, lens, bounds)
    with pytest.raises(ValueError, match="must be CUDA tensors"):
        fd.paged_block_select(q, k, bounds, table, lens, 4)
    selection = fd.BlockSelection(*(torch.zeros(s, dtype=torch.int32) for s in ((2, 2, 3), (2, 2, 3), (2, 2))), 2)
    with pytest.raises(ValueError, match="must be CUDA tensors"):
        fd.paged_decode_attention_blocks(q, k, v, selection)
    for bad in (None, 3, [1]):
        with pytest.raises(TypeError, match="must be a torch.Tensor"):
            fd.paged_key_bounds(bad, table, lens, bounds)
        with pytest.raises(TypeError, match="must be a torch.Tensor"):
            fd.paged_block_select(bad, k, bounds, table, lens, 4)
        with pytest.raises(TypeError, match="must be a torch.Tensor"):
            fd.paged_decode_attention_blocks(bad, k, v, selection)
    for cache, tables in ((k[0], table), (k, table[0]), (k[0, 0, 0], table), (k, lens[0]), (k.byte(), table)):
        with pytest.raises(ValueError, match="must be a 2D tensor"):
            fd.paged_block_select(q, cache, bounds, tables, lens, 4)
    with pytest.raises(TypeError, match="BlockSelection"):
        fd.paged_decode_attention_blocks(q, k, v, (1, 2, 3, 4))


def _filled(kind, **over):
    a = kind(dtype=_lib.FD_DTYPE_BF16, num_seqs=2, num_kv_heads=2, head_dim=128, block_size=32, num_blocks=4,
             max_blocks_per_seq=3, block_tables=16, seq_lens=16, bounds=16)
    if kind is _lib.KeyBoundsArgs:
        a.k_cache, a.new_tokens = 16, 1
    else:
        a.num_q_heads, a.q, a.select, a.sink_blocks, a.recent_blocks, a.block_step = 4, 16, 2, 1, 1, 2
        a.blocks, a.tables, a.lens = 16, 16, 16
    a.struct_size = ctypes.sizeof(a)
    for name, value in over.items():
        setattr(a, name, value)
    return a


def test_the_library_refuses_bad_arguments():
    """Pointers that are never dereferenced: every call is refused before any HIP call."""
    lib = _lib.load_library()
    big, words = 1 << 62, ctypes.c_int64()
    shared = ((dict(struct_size=8), b"struct_size"), (dict(dtype=_lib.FD_DTYPE_F32), b"dtype"), (dict(head_dim=96), b"head_dim"),
              (dict(block_size=64), b"block_size"), (dict(num_seqs=0), b"positive"), (dict(num_seqs=big), b"grid"),
              (dict(num_kv_heads=-1), b"positive"), (dict(num_blocks=0), b"positive"), (dict(num_blocks=big), b"too many"),
              (dict(max_blocks_per_seq=0), b"positive"), (dict(max_blocks_per_seq=big), b"2^31 tokens"),
              (dict(max_blocks_per_seq=1 << 26), b"2^31 tokens"), (dict(bounds=None), b"NULL"), (dict(bounds=24), b"aligned"),
              (dict(block_tables=None), b"NULL"), (dict(seq_lens=None), b"NULL"))
    for over, message in (*shared, (dict(k_cache=None), b"NULL"), (dict(new_tokens=-1), b"new_tokens")):
        assert lib.fd_key_bounds(ctypes.byref(_filled(_lib.KeyBoundsArgs, **over)), None) < 0, over
        assert message in lib.fd_last_error(), (over, lib.fd_last_error())
    assert lib.fd_key_bounds(None, None) < 0
    assert lib.fd_key_bounds(ctypes.byref(_filled(_lib.KeyBoundsArgs, new_tokens=0)), None) == 0
    for over, message in (
            *shared, (dict(num_q_heads=3), b"divisible"), (dict(num_q_heads=0), b"divisible"), (dict(select=0), b"select"),
            (dict(select=big), b"select"), (dict(sink_blocks=-1), b"select"), (dict(recent_blocks=0), b"select"),
            (dict(sink_blocks=2), b"select"), (dict(sink_blocks=big, recent_blocks=big), b"select"),
            (dict(block_step=1), b"32-bit"), (dict(block_step=big), b"32-bit"), (dict(num_blocks=1 << 30), b"32-bit"),
            (dict(q=None), b"NULL"), (dict(blocks=None), b"NULL"), (dict(tables=None), b"NULL"), (dict(lens=None), b"NULL"),
            (dict(num_seqs=40000), b"grid")):
        args = _filled(_lib.BlockSelectArgs, **over)
        assert lib.fd_block_select_words(ctypes.byref(args), ctypes.byref(words)) < 0, over
        assert message in lib.fd_last_error(), (over, lib.fd_last_error())
        assert lib.fd_block_select(ctypes.byref(args), None, 0, None) < 0, over
        assert message in lib.fd_last_error(), (over, lib.fd_last_error())
    good = _filled(_lib.BlockSelectArgs)
    assert lib.fd_block_select_words(ctypes.byref(good), ctypes.byref(words)) == 0 and words.value == 12
    assert lib.fd_block_select_words(ctypes.byref(good), None) < 0 and lib.fd_block_select_words(None, None) < 0
    for workspace, n in ((None, 12), (16, 11), (17, 12)):
        assert lib.fd_block_select(ctypes.byref(good), workspace, n, None) < 0 and b"workspace" in lib.fd_last_error()


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_structs_match_the_c_layout(tmp_path):
    pairs = [("fd_key_bounds_args", _lib.KeyBoundsArgs), ("fd_block_select_args", _lib.BlockSelectArgs)]
    src = tmp_path / "probe.c"
    lines = "".join(f'  printf("%zu\\n", sizeof({c}));\n' + "".join(f'  printf("%zu\\n", offsetof({c}, {f}));\n'
                                                                   for f, _ in s._fields_) for c, s in pairs)
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "flashdec_hip.h"\nint main(void) {\n' + lines
                   + "  return 0;\n}\n")
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", str(HEADER.parent), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    want = [x for _, s in pairs for x in (ctypes.sizeof(s), *(getattr(s, f).offset for f, _ in s._fields_))]
    assert got == want


def test_names_are_exported():
    for name in ("BlockSelection", "paged_key_bounds", "paged_block_select", "paged_block_select_into",
                 "paged_decode_attention_blocks", "paged_decode_attention_blocks_into"):
        assert name in fd.__all__ and getattr(fd, name) is getattr(sparse, name)


def test_lists_that_hold_the_whole_table_need_no_workspace():
    lib, words = _lib.load_library(), ctypes.c_int64(-1)
    for select, width, want in ((3, 3, 0), (100, 3, 0), (2, 3, 12), (3, 4, 16), (3, 5000, 20000), (5000, 5000, 0)):
        args = _filled(_lib.BlockSelectArgs, select=select, max_blocks_per_seq=width)
        assert lib.fd_block_select_words(ctypes.byref(args), ctypes.byref(words)) == 0 and words.value == want
