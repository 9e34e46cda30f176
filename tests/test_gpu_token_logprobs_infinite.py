"""Infinite logits under infinite temperatures: token_logprobs_f32 on the GPU against the
plain 64-bit form (tests/serving_oracle.py)."""
import math

import numpy as np
import pytest

from test_gpu_token_logprobs import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [5, 300, 9000])
@pytest.mark.parametrize("temperature", [math.inf, 3.4e38, 1.0, 1e-45])
def test_a_logit_below_an_infinite_one_has_no_share(hip_ctx, size, temperature):
    rng = np.random.default_rng(size)
    rows = rng.standard_normal((4, size))
    rows[0, size // 2] = math.inf
    rows[1, [0, size - 1]] = math.inf
    rows[2, 1:4] = (math.inf, -math.inf, math.nan)
    rows[3, :3] = (3.4e38, -3.4e38, -math.inf)  # (finite: all real logits alike at infinity)
    for tokens in ([0] * 4, [size - 1] * 4, [size // 2] * 4, [1, 2, 3, 1], [2, 1, 2, 2]):
        got = check(hip_ctx, rows, tokens, 5, [temperature] * 4)
        for n in ("logprob", "entropy", "top_logprobs"):
            assert not np.isnan(got[n]).any(), n
