"""The 4-bit cache on the CPU: the format, its plain forms, and every refusal before a launch."""

import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import flashdec_amd as fd
from flashdec_amd import _lib, fp4
from flashdec_amd.bounded import _apart
from tests import fp4_oracle as fo

HEADER = Path(__file__).resolve().parents[1] / "include" / "flashdec_hip.h"


def test_block_bytes():
    assert fd.fp4_block_bytes(32, 128) == 2176 and fd.fp4_block_bytes(8, 64) == 272
    for bad in ((4, 128), (64, 128), (32, 96), (32, 0), (True, 128)):
        with pytest.raises(ValueError, match="4-bit cache supports"):
            fd.fp4_block_bytes(*bad)


@pytest.mark.parametrize("block", [8, 16, 32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("values", [False, True])
def test_a_block_holds_each_code_and_scale_once(block, d, values):
    code_at, shift, scale_at = fo.places(block, d, values)
    taken = torch.cat(((2 * code_at + shift // 4).flatten(), (2 * scale_at).flatten(), (2 * scale_at + 1).flatten()))
    assert torch.equal(taken.sort().values, torch.arange(2 * fo.block_bytes(block, d)))


def test_scales_leave_every_value_within_half_of_its_step():
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(4000, 32, generator=gen, dtype=torch.float64).float() * torch.exp2(torch.randint(-30, 30, (4000, 1),
                                                                                               generator=gen).float())
    codes, byte = fo.quantise(x)
    unit = torch.exp2(byte.double() - 127)
    got = fo.LEVELS[codes % 8] * torch.where(codes >= 8, -1.0, 1.0) * unit
    a = x.double().abs() / unit
    assert float(a.max()) <= 7 and float(a.amax(dim=1).min()) > 3.5
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    assert bool(((got - x.double()).abs() <= step / 2 * unit).all())


def test_edges_of_the_format():
    x = torch.zeros(6, 32)
    x[1, 3] = math.nan
    x[2, 0], x[2, 1] = math.inf, 1.0
    x[3, 0] = 3.3e38
    x[4, 0] = 1e-44
    x[5, :6] = torch.tensor([7.0, 5.0, 2.5, -0.25, 0.75, -3.5])
    codes, byte = fo.quantise(x)
    assert byte.flatten().tolist() == [2, 255, 255, 252, 2, 127]
    assert codes[0].sum() == 0 and codes[3, 0] == 7 and codes[4, 0] == 0
    assert codes[5, :6].tolist() == [7, 6, 4, 8, 2, 14]


def test_rotary_settings_and_tensors_are_refused_on_the_cpu():
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    pool = torch.zeros(4, 2, fo.block_bytes(16, 64), dtype=torch.uint8)
    at = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        fd.kv_append_fp4(k, k, pool, pool.clone(), at, at)
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        fd.fused_rope_kv_append_fp4(k, k, k, pool, pool.clone(), at, at, at)
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        fd.paged_kv_read_fp4(pool, pool.clone(), at, at, 64)
    for bad in (None, 3, [1]):
        with pytest.raises(TypeError, match="must be a torch.Tensor"):
            fd.kv_append_fp4(bad, k, pool, pool.clone(), at, at)
        with pytest.raises(TypeError, match="must be a torch.Tensor"):
            fd.paged_kv_read_fp4_into(pool, pool, at, at, bad, k)


class _OnGpu(torch.Tensor):
    """A CPU tensor that says it is on a GPU: the checks run, no launch does."""

    @property
    def is_cuda(self):
        return True


def _fake(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype).as_subclass(_OnGpu)


def _append(**over):
    t = {"q": _fake(3, 4, 64), "k": _fake(3, 2, 64), "v": _fake(3, 2, 64),
         "k_cache": _fake(5, 2, fo.block_bytes(16, 64), dtype=torch.uint8),
         "v_cache": _fake(5, 2, fo.block_bytes(16, 64), dtype=torch.uint8),
         "block_ids": _fake(3, dtype=torch.int64), "block_offsets": _fake(3, dtype=torch.int32),
         "positions": _fake(3, dtype=torch.int64), "rotary_dim": 64, "base": 10000.0, "table": None, "q_out": None}
    t.update(over)
    return fp4._append_args(t["q"], t["k"], t["v"], t["k_cache"], t["v_cache"], t["block_ids"], t["block_offsets"],
                            t["positions"], t["rotary_dim"], t["base"], t["table"], t["q_out"])


def test_append_checks():
    args = _append()
    assert (args.num_tokens, args.block_size, args.num_blocks, list(args.index_dtype)) == (3, 16, 5, [1, 0, 1])
    assert _append(rotary_dim=20, q=_fake(3, 12, 64)[:, ::3], k=_fake(6, 2, 64)[::2]).rotary_dim == 20
    nb = fo.block_bytes(16, 64)
    planes = _fake(5, 2, 2, nb, dtype=torch.uint8)  # K and V of a block next to each other
    assert list(_append(k_cache=planes[:, 0], v_cache=planes[:, 1]).k_cache_stride) == [4 * nb, nb]
    u8 = torch.uint8
    for over, message in (
            (dict(k=_fake(3, 2, 64, dtype=torch.float32)), "float16 and bfloat16"),
            (dict(k=_fake(3, 128)), "shape"), (dict(v=_fake(3, 1, 64)), "shape"), (dict(v=_fake(2, 2, 64)), "shape"),
            (dict(v=_fake(3, 2, 64, dtype=torch.float16)), "same dtype"), (dict(k=_fake(3, 64, 2).transpose(1, 2)), "unit dim"),
            (dict(k=_fake(3, 3, 64), v=_fake(3, 3, 64)), "num_kv_heads"), (dict(q=_fake(4, 4, 64)), "shape"),
            (dict(q=_fake(3, 0, 64)), "num_q_heads"), (dict(k_cache=_fake(5, 2, nb)), "uint8"),
            (dict(k_cache=_fake(5, 2, nb, 1, dtype=u8)), "uint8"), (dict(k_cache=_fake(4, 2, nb, dtype=u8)), "same shape"),
            (dict(k_cache=_fake(0, 2, nb, dtype=u8), v_cache=_fake(0, 2, nb, dtype=u8)), "positive"),
            (dict(k_cache=_fake(5, 2, nb + 16, dtype=u8), v_cache=_fake(5, 2, nb + 16, dtype=u8)), "fp4_block_bytes"),
            (dict(k_cache=_fake(5, 2, 4, dtype=u8), v_cache=_fake(5, 2, 4, dtype=u8)), "fp4_block_bytes"),
            (dict(k_cache=_fake(5, 2, nb + 8, dtype=u8)[..., :nb]), "16-byte lines"),
            (dict(k_cache=_fake(5, 2, 2 * nb, dtype=u8)[..., ::2]), "16-byte lines"),
            (dict(k_cache=_fake(1, 2, nb, dtype=u8).expand(5, 2, nb)), "overlapping"),
            (dict(block_ids=_fake(2, dtype=torch.int64)), "one value per token"),
            (dict(block_ids=_fake(3, dtype=torch.int16)), "int32 or int64"),
            (dict(block_offsets=_fake(6, dtype=torch.int32)[::2]), "contiguous"),
            (dict(positions=_fake(3, 1, dtype=torch.int64)), "one value per token"),
            (dict(rotary_dim=63), "even"), (dict(rotary_dim=66), "even"), (dict(rotary_dim=0), "even"),
            (dict(rotary_dim=True), "integer"), (dict(rotary_dim=32.0), "integer"), (dict(base=math.inf), "base"),
            (dict(base=-1.0), "base"), (dict(table=_fake(2, 9, 16, dtype=torch.float32)), "cos_sin_table"),
            (dict(q_out=_fake(3, 3, 64)), "shape"), (dict(q_out=_fake(3, 1, 64).expand(3, 4, 64)), "overlapping"),
            (dict(k=_fake(3, 2, 96), v=_fake(3, 2, 96)), "head_dim")):
        with pytest.raises((ValueError, TypeError), match=message):
            _append(**over)


def test_read_checks():
    nb = fo.block_bytes(8, 128)
    pool, at, out = _fake(5, 2, nb, dtype=torch.uint8), _fake(3, dtype=torch.int64), _fake(3, 2, 128)
    assert fp4._read_args(pool, pool, at, at, out, _fake(3, 2, 128)).block_size == 8
    for args, message in (((pool, pool, at, at, out.float(), out), "float16 or bfloat16"),
                          ((pool, pool, at, at, out, out.half()), "same dtype"),
                          ((pool, pool, at, at[:2], out, out), "one value per token"),
                          ((pool, pool, at, at, out, _fake(3, 1, 128).expand(3, 2, 128)), "overlapping"),
                          ((pool, pool, at, at, _fake(3, 3, 128), _fake(3, 3, 128)), "num_kv_heads")):
        with pytest.raises(ValueError, match=message):
            fp4._read_args(*args)


def _c_append(**over):
    a = _lib.Fp4AppendArgs(dtype=_lib.FD_DTYPE_BF16, num_tokens=2, num_q_heads=4, num_kv_heads=2, head_dim=128, block_size=32,
                           num_blocks=4, rotary_dim=128, base=1e4, q=16, k=16, v=16, q_out=16, k_cache=16, v_cache=32,
                           block_ids=16, block_offsets=16, positions=16)
    a.struct_size = ctypes.sizeof(a)
    for name, value in over.items():
        if isinstance(value, tuple):
            getattr(a, name)[:] = value
        else:
            setattr(a, name, value)
    return a


def test_the_library_refuses_bad_append_and_read_arguments():
    """Pointers that are never dereferenced: every call is refused before any HIP call."""
    lib = _lib.load_library()
    big = 1 << 62
    for over, message in (
            (dict(struct_size=8), b"struct_size"), (dict(dtype=_lib.FD_DTYPE_F32), b"dtype"), (dict(head_dim=96), b"head_dim"),
            (dict(block_size=64), b"block_size"), (dict(num_blocks=0), b"positive"), (dict(num_blocks=big), b"too many"),
            (dict(num_kv_heads=-1), b"positive"), (dict(num_kv_heads=big), b"too many"), (dict(num_tokens=-1), b"positive"),
            (dict(num_tokens=big), b"grid"), (dict(k_cache=None), b"NULL"), (dict(k_cache=24), b"aligned"),
            (dict(k_cache_stride=(8, 0)), b"strides"), (dict(v_cache_stride=(0, -16)), b"strides"), (dict(k=None), b"NULL"),
            (dict(block_ids=None), b"NULL"), (dict(q=None), b"rotation"), (dict(q_out=None), b"rotation"),
            (dict(positions=None), b"rotation"), (dict(num_q_heads=0), b"rotation"), (dict(num_q_heads=big), b"query heads"),
            (dict(rotary_dim=-2), b"rotary_dim"), (dict(rotary_dim=130), b"rotary_dim"), (dict(rotary_dim=7), b"rotary_dim"),
            (dict(base=0.0), b"base"), (dict(base=math.nan), b"base"), (dict(cos_sin_table=16), b"table_rows"),
            (dict(cos_sin_table=18, table_rows=4), b"table_rows")):
        assert lib.fd_fp4_append(ctypes.byref(_c_append(**over)), None) < 0, over
        assert message in lib.fd_last_error(), (over, lib.fd_last_error())
    assert lib.fd_fp4_append(None, None) < 0 and lib.fd_fp4_read(None, None) < 0
    assert lib.fd_fp4_append(ctypes.byref(_c_append(num_tokens=0)), None) == 0

    def read(**over):
        a = _lib.Fp4ReadArgs(dtype=_lib.FD_DTYPE_F16, num_tokens=2, num_kv_heads=2, head_dim=64, block_size=8, num_blocks=4,
                             k_cache=16, v_cache=32, block_ids=16, block_offsets=16, k_out=16, v_out=16)
        a.struct_size = ctypes.sizeof(a)
        for name, value in over.items():
            setattr(a, name, value)
        return a

    for over, message in ((dict(struct_size=8), b"struct_size"), (dict(dtype=_lib.FD_DTYPE_F32), b"dtype"),
                          (dict(num_tokens=-1), b"positive"), (dict(num_tokens=big), b"grid"), (dict(v_out=None), b"NULL"),
                          (dict(num_tokens=1 << 24, num_kv_heads=65535), b"grid"), (dict(v_cache=8), b"aligned")):
        assert lib.fd_fp4_read(ctypes.byref(read(**over)), None) < 0, over
        assert message in lib.fd_last_error(), (over, lib.fd_last_error())
    assert lib.fd_fp4_read(ctypes.byref(read(num_tokens=0)), None) == 0


def _c_decode(**over):
    a = _lib.Fp4DecodeArgs(dtype=_lib.FD_DTYPE_BF16, num_seqs=2, num_q_heads=4, num_kv_heads=2, head_dim=128, block_size=32,
                           num_blocks=4, max_blocks_per_seq=3, q=16, k_cache=16, v_cache=32, block_tables=16, seq_lens=16,
                           out=16, sm_scale=0.1)
    a.struct_size = ctypes.sizeof(a)
    for name, value in over.items():
        if isinstance(value, tuple):
            getattr(a, name)[:] = value
        else:
            setattr(a, name, value)
    return a


def test_the_library_refuses_bad_decode_arguments():
    lib = _lib.load_library()
    big, floats = 1 << 62, ctypes.c_int64()
    for over, message in (
            (dict(struct_size=8), b"struct_size"), (dict(dtype=_lib.FD_DTYPE_F32), b"dtype"), (dict(head_dim=96), b"head_dim"),
            (dict(block_size=4), b"block_size"), (dict(num_seqs=0), b"positive"), (dict(num_seqs=65536), b"grid"),
            (dict(num_seqs=big), b"grid"), (dict(num_q_heads=0), b"positive"), (dict(num_q_heads=3), b"divisible"),
            (dict(num_q_heads=big), b"grid"), (dict(num_kv_heads=65536, num_q_heads=65536), b"too many"),
            (dict(max_blocks_per_seq=0), b"positive"), (dict(max_blocks_per_seq=1 << 31), b"2^31 tokens"),
            (dict(max_blocks_per_seq=(1 << 31) // 32), b"2^31 tokens"), (dict(max_blocks_per_seq=big), b"2^31 tokens"),
            (dict(num_blocks=big), b"too many"), (dict(q=None), b"NULL"), (dict(out=None), b"NULL"),
            (dict(seq_lens=None), b"NULL"), (dict(block_tables=None), b"NULL"), (dict(seq_lens_stride=-1), b"stride"),
            (dict(seq_lens_stride=1 << 31), b"stride"), (dict(k_cache=8), b"aligned"), (dict(v_cache_stride=(8, 0)), b"strides"),
            (dict(kv_reuse=2), b"0 or 1"), (dict(ragged=-1), b"0 or 1")):
        args = _c_decode(**over)
        assert lib.fd_fp4_decode_floats(ctypes.byref(args), ctypes.byref(floats)) < 0, over
        assert message in lib.fd_last_error(), (over, lib.fd_last_error())
        assert lib.fd_fp4_decode(ctypes.byref(args), None, 0, None) < 0, over
        assert message in lib.fd_last_error(), (over, lib.fd_last_error())
    assert lib.fd_fp4_decode(None, None, 0, None) < 0 and lib.fd_fp4_decode_floats(None, ctypes.byref(floats)) < 0
    assert lib.fd_fp4_decode_floats(ctypes.byref(_c_decode()), None) < 0


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_structs_match_the_c_layout(tmp_path):
    pairs = [("fd_fp4_append_args", _lib.Fp4AppendArgs), ("fd_fp4_read_args", _lib.Fp4ReadArgs),
             ("fd_fp4_decode_args", _lib.Fp4DecodeArgs)]
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
    for name in ("fp4_block_bytes", "fused_rope_kv_append_fp4", "kv_append_fp4", "paged_kv_read_fp4",
                 "paged_kv_read_fp4_into", "paged_decode_attention_fp4", "paged_decode_attention_fp4_into"):
        assert name in fd.__all__ and getattr(fd, name) is getattr(fp4, name)


def test_tensors_that_lie_apart():
    """What is said to be apart shares no element; slices of one buffer, by tokens, heads or dims, are seen to be."""
    buffer = torch.zeros(6, 10, 24)
    places = torch.arange(buffer.numel()).view_as(buffer)

    def held(t):
        return set(places.as_strided(t.shape, t.stride(), t.storage_offset()).flatten().tolist())

    turned = buffer.as_strided((10, 6, 24), (24, 240, 1))
    views = [buffer, buffer[:3], buffer[3:], buffer[::2], buffer[1::2], buffer[:, :4], buffer[:, 4:], buffer[:, 3:7],
             buffer[:, ::2], buffer[:, 1::2], buffer[..., :8], buffer[..., 8:], buffer[..., 6:20], buffer[1:2, 2:3],
             turned[:4], turned[4:], turned[::3], turned[:, :, 8:], buffer[:, :1].expand(6, 10, 24), buffer[2, 3:4, 5:6],
             buffer[5:, 9:, 23:], buffer.as_strided((4, 5, 3), (17, 29, 5), 11)]
    gen = torch.Generator().manual_seed(3)
    for _ in range(60):
        shape = torch.randint(1, 5, (3,), generator=gen).tolist()
        stride = torch.randint(0, 90, (3,), generator=gen).tolist()
        views.append(buffer.as_strided(shape, stride, int(torch.randint(0, 300, (1,), generator=gen))))
    for a in views:
        for b in views:
            assert not (_apart(a, b) and held(a) & held(b))
    for a, b in ((views[1], views[2]), (views[3], views[4]), (views[5], views[6]), (views[8], views[9]), (views[10], views[11]),
                 (views[14], views[15]), (views[10], views[17]), (views[5], views[15]), (views[13], views[19])):
        assert _apart(a, b) and _apart(b, a)
    assert _apart(buffer[:0], buffer) and not _apart(buffer, buffer)


@pytest.mark.parametrize("bad", [None, 3, [1]])
def test_a_query_that_is_no_tensor_is_refused(bad):
    k, at = _fake(3, 2, 64), _fake(3, dtype=torch.int64)
    pools = [_fake(5, 2, fo.block_bytes(16, 64), dtype=torch.uint8) for _ in range(2)]
    for rotary in (None, 64):
        with pytest.raises(TypeError, match="q must be a torch.Tensor"):
            fd.fused_rope_kv_append_fp4(bad, k, k, *pools, at, at, at, rotary_dim=rotary)
