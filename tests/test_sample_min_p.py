"""CPU tests of the sampling call with options per row: what it refuses, before any device is
touched, and the plain implementation the GPU tests compare with, on rows small enough to check
by hand."""
import ctypes
import math

import numpy as np
import pytest

from neuraval_b200 import native
from neuraval_b200.sampler import sample_rows_min_p_device
from tests.min_p_ref import sample_row

GOOD = dict(logits=0x1000, dtype=native.DTYPE_F32, rows=2, vocab=8, ld=8, uniforms=0x2000,
            temperature=None, top_k=None, top_p=None, min_p=None, tokens=0x3000, logprobs=None,
            kept=None, flags=None, stream=None)


def call(navlib, **over):
    a = dict(GOOD, **over)
    return navlib.ncb_sample_rows_min_p_device(*a.values())


@pytest.mark.parametrize("over", [
    dict(logits=None), dict(uniforms=None), dict(tokens=None), dict(dtype=3), dict(dtype=-1),
    dict(rows=-1), dict(vocab=0), dict(vocab=-5), dict(ld=7), dict(logits=0x1002),
    dict(logits=0x1001, dtype=native.DTYPE_BF16), dict(uniforms=0x2002), dict(top_k=0x4001),
    dict(flags=0x5002), dict(logprobs=0x5003), dict(kept=0x5001), dict(min_p=0x5001),
], ids=str)
def test_refused_arguments(navlib, over):
    assert call(navlib, **over) == native.NCB_ERROR_INVALID_ARGUMENT
    assert navlib.ncb_sampler_last_status() == native.NCB_ERROR_INVALID_ARGUMENT


def test_capacity_and_empty_batch(navlib):
    assert call(navlib, vocab=(1 << 24) + 1, ld=1 << 25) == native.NCB_ERROR_CAPACITY
    assert call(navlib, rows=0, logits=None, uniforms=None, tokens=None) == native.NCB_OK


def test_front_end_refuses(navlib):
    import torch
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError):
        sample_rows_min_p_device(x, torch.zeros(2), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        sample_rows_min_p_device(x[0], torch.zeros(2), torch.zeros(2, dtype=torch.int32))


def test_plain_implementation_by_hand():
    x = [0.0, math.log(4.0), -math.inf, math.log(2.0), math.log(2.0)]  # weights .25 1 - .5 .5
    assert sample_row(x, 0.0, 0, 1.0, 0.0, 0.9) == (1, 1, 0.0)
    # all: order 1 3 4 0, masses 1 1.5 2 2.25
    assert [sample_row(x, 1.0, 0, 1.0, 0.0, u)[0] for u in (0.0, 0.44, 0.45, 0.67, 0.99)] == \
        [1, 1, 3, 4, 0]
    assert sample_row(x, 1.0, 2, 1.0, 0.0, 0.7)[:2] == (3, 2)  # equal values: the lower id first
    assert sample_row(x, 1.0, 0, 0.5, 0.0, 0.99)[:2] == (3, 2)  # 1 < 0.5 * 2.25 <= 1.5
    assert sample_row(x, 1.0, 0, 1.0, 0.4, 0.99)[:2] == (4, 3)
    tok, n, lp = sample_row(x, 1.0, 3, 0.99, 0.3, 0.0)
    assert (tok, n) == (1, 3) and abs(lp - math.log(0.5)) < 1e-15
    assert np.isfinite(lp)


def test_abi_signature_matches_header(navlib):
    assert ctypes.sizeof(ctypes.c_int64) == 8
    assert len(native.SIGNATURES["ncb_sample_rows_min_p_device"][1]) == len(GOOD)
