"""What a sequence or a row gets in a batch, and by itself: key weights to their tolerance (a
batch's number of sequences and bounds choose how keys and rows are cut), log probabilities to
the bit (a row's cut goes by its size alone)."""
import numpy as np
import pytest

import paged_oracle as po
import serving_oracle as so
from test_gpu_key_weights import run as run_weights
from test_gpu_paged_q8 import Batch
from test_gpu_token_logprobs import run as run_logprobs

pytestmark = pytest.mark.gpu


def alone(rng, batch, b, page_tokens):
    """Sequence b of a batch as a batch of its own, over the same pages."""
    one = Batch(rng, page_tokens, [batch.new[b]], [batch.before[b]])
    one.table[:] = batch.table[b:b + 1, :one.width]
    return one


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new,before", [([1, 2, 1, 1], [900, 33, 4000, 64]),  # few rows each
                                        ([1, 40, 3, 300], [500, 300, 20, 1000])])
def test_key_weights_of_a_sequence_alone(hip_ctx, new, before, f16):
    rng = np.random.default_rng(sum(before))
    batch = Batch(rng, 16, new, before)
    cache = po.Pages(rng, batch.pages, 16, 2, 128)
    query = (2 * rng.standard_normal((batch.tokens, 4, 128))).astype(np.float16 if f16 else np.float32)
    stride = int(batch.lengths.max()) + 5
    old = rng.random((len(new), 2, stride)).astype(np.float32)
    whole = run_weights(hip_ctx, cache, batch, 4, query, old, 0, 0.5)
    np.testing.assert_array_equal(whole, run_weights(hip_ctx, cache, batch, 4, query, old, 0, 0.5))
    for b in range(len(new)):
        one = alone(rng, batch, b, 16)
        mine = query[int(batch.starts[b]):int(batch.starts[b + 1])]
        got = run_weights(hip_ctx, cache, one, 4, mine, old[b:b + 1], 0, 0.5)
        want, tol = so.key_weights(cache, mine, one.plain(), 4, 0, 0.5, old[b:b + 1], stride)
        # (Each is within its tolerance of the definition's.)
        assert (np.abs(got - want) <= tol).all()
        assert (np.abs(whole[b:b + 1] - want) <= tol).all()
        assert (np.abs(got - whole[b:b + 1].astype(np.float64)) <= 2 * tol).all()


@pytest.mark.parametrize("size", [900, 4096, 20000, 70001])
def test_log_probabilities_of_a_row_alone(hip_ctx, size):
    rng = np.random.default_rng(size)
    logits = (3 * rng.standard_normal((40, size))).astype(np.float32)
    tokens = rng.integers(0, size, 40)
    temperature = rng.choice([0.5, 1.0, 1.7], 40)
    whole = run_logprobs(hip_ctx, logits, tokens, 20, temperature)
    for r in (0, 17, 38, 39):
        one = run_logprobs(hip_ctx, logits[r:r + 1], tokens[r:r + 1], 20, temperature[r:r + 1])
        assert len(one) == 5
        for n, x in one.items():
            np.testing.assert_array_equal(x[0], whole[n][r], err_msg=n)
