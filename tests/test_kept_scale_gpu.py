"""Calls that repeat take the last one's arguments: the scale's value at each call counts, whatever object holds it."""

import pytest
import torch

from oracle.attention import paged_decode_attention as oracle_decode
from tests.helpers import assert_close_to_oracle, make_paged_inputs, np32

pytestmark = pytest.mark.gpu


def _holders():
    import numpy as np

    return np.zeros(()), torch.zeros(())


def _check(out, q, k, v, table, lens, scale):
    want = oracle_decode(np32(q), np32(k), np32(v), table.cpu().numpy(), lens.cpu().numpy(), sm_scale=scale)
    assert_close_to_oracle(out, want)


def test_decode():
    import flashdec_amd as fd

    case = make_paged_inputs([600, 40], 16, 2, 128, 32, seed=3)
    for ragged in (False, True):
        for scale in _holders():
            for value in (0.05, 0.3, -0.1, 0.05):
                scale[...] = value
                _check(fd.decode(*case, sm_scale=scale, ragged=ragged), *case, float(scale))


def test_cascade():
    from flashdec_amd import cascade

    q, k, v, table, lens = make_paged_inputs([600, 530, 700], 16, 2, 128, 32, seed=4)
    table[1:, :16] = table[0, :16]
    groups = cascade.build_cascade_groups(table, lens, block_size=32, num_q_heads=16, num_kv_heads=2)
    assert groups is not None
    out = torch.empty_like(q)
    for scale in _holders():
        for value in (0.05, 0.3, -0.1, 0.05):
            scale[...] = value
            cascade.paged_decode_attention_cascade_into(q, k, v, table, lens, out, groups, sm_scale=scale)
            _check(out, q, k, v, table, lens, float(scale))
