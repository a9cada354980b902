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
