"""sample_f32_i32 where logits and temperature lie at the ends of f32's range, with the
tolerances of tests/test_gpu_sample.py."""
import numpy as np
import pytest

from test_gpu_sample import check

pytestmark = pytest.mark.gpu

UNIFORMS = [0.0, 0.3, 0.6, 0.9, 0.99, 0.9999]


@pytest.mark.parametrize("rules", [{}, {"min_p": 0.01}, {"min_p": 0.3}, {"min_p": 0.01, "top_k": 9},
                                   {"top_p": 0.95}, {"top_p": 0.9, "top_k": 40, "min_p": 1e-3}])
@pytest.mark.parametrize("top,low,temperature", [
    (3e38, -3e38, 1e38),  # differences that f32 does not hold
    (3.4e38, -1e38, 7e37),
    (1e-38, -1e-38, 4e-39),  # 1 / T beyond f32's largest
    (4e-44, -4e-44, 3e-44),  # steps of the least subnormal
])
def test_logits_at_the_ends_of_the_range(hip_ctx, top, low, temperature, rules):
    rng = np.random.default_rng(71)
    rows, size = len(UNIFORMS), 3000
    x = rng.uniform(low, top, (rows, size)).astype(np.float32)
    x[:, rng.permutation(size)[:2900]] = np.float32(low)
    x[:, 17] = top
    # (The f32 number, for both sides.)
    check(hip_ctx, x, np.array(UNIFORMS, np.float32), temperature=[np.float32(temperature)] * rows,
          **{n: [v] * rows for n, v in rules.items()})
