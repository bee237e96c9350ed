"""The quotient by the repetition penalty in ku_hip_logits_adjust: correctly rounded, over the whole range of f32."""
import numpy as np
import pytest

from kurumi_amd import DType
from test_gpu_logits_adjust import call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [3, 300], ids=["few rows", "many rows"])
def test_the_quotient_is_rounded_once(hip, rows):
    """y = x / repetition for positive x that was seen, x * repetition for others: each one f32 operation."""
    rng = np.random.default_rng(rows)
    vocab = 8200
    x = (rng.standard_normal((rows, vocab)) * 2.0 ** rng.integers(-20, 20, (rows, vocab))).astype(np.float32)
    rep = (1 + rng.random(rows)).astype(np.float32)
    rep[0], rep[1] = np.float32(2) - np.float32(2.0 ** -23), np.float32(1.3)  # every bit of its significand; a common one
    tokens = np.tile(np.arange(vocab, dtype=np.int32), (rows, 1))
    got = call(hip, x, DType.F32, DType.F32, tokens=tokens, rep=rep)
    want = np.where(x > 0, x / rep[:, None], x * rep[:, None])
    np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("rep", [2.0 ** -149, 1e-39, 2.0 ** -127, 2.0 ** -126 * 1.7, 1e-30, 1e30, 3e38, float(np.finfo(np.float32).max), np.inf])
def test_penalties_and_logits_of_every_size(hip, rep):
    """A penalty whose reciprocal is past the largest f32, or under the smallest normal one, has finite quotients."""
    rep = np.float32(rep)
    x = np.array([[2.0 ** -149, 1e-42, 3e-39, 2.0 ** -126, 1.1e-38, 7e-31, 1.0, 3.3, 1e10, 1e37, 3.3e38, np.inf, 0.0, -0.0, np.nan, -1.5, -1e-40, -1e38]],
                 np.float32)
    with np.errstate(all="ignore"):
        want = np.where(x > 0, x / rep, x * rep)
    got = call(hip, x, DType.F32, DType.F32, tokens=np.arange(x.shape[1], dtype=np.int32)[None], rep=np.array([rep]))
    np.testing.assert_array_equal(got, want)
