"""Sampling with options per row where its searches have little to go by: a least value that min-p
keeps next to 0. Against the definition in 64 bits; the values stand off the borders by more than
64-bit rounding."""
import math

import numpy as np
import pytest

from tests.test_sample_min_p_gpu import compare, dtype_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_least_kept_value_next_to_zero(dtype):
    """max + T ln min_p cancels to nothing: all tiny values are as far from the maximum."""
    import torch
    rng = np.random.default_rng(1)
    rows = []  # maximum, T, min_p
    if dtype == "f32":
        rows += [(1.83644283, 0.802564383, 0.101447009), (3.73568249, 0.967938006, 0.0210801531)]
    rows += [(mx, T, math.exp(-mx / T)) for mx, T in ((2.0, 1.0), (1.5, 0.75), (6.0, 1.25), (0.5, 0.3))]
    n = len(rows)
    x = rng.choice(np.array([-3.0, -0.01, 0.01, 0.25]), (2 * n, 4099))
    x[:, 17] = [r[0] for r in rows] * 2
    opt = np.array(rows * 2)
    # once with min-p alone, once with a top-k and a top-p that need the exact passes
    compare(torch.from_numpy(x).cuda().to(dtype_of(dtype)), opt[:, 1], [0] * n + [3000] * n,
            [1.0] * n + [0.99] * n, opt[:, 2], rng.random(2 * n))
