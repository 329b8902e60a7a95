"""Attention of keys whose scores are equal or opposite: the exact weights are known at
any size of score, so that what a score's rounding costs is not part of the bounds."""
import numpy as np
import pytest

from tests import attention_oracle as oracle
from tests.attention_oracle import assert_within, half_step
from tests.test_attention_gpu import F32, F64, _release_buffers, attend  # noqa: F401

pytestmark = pytest.mark.gpu

SHAPES = [  # (batch, heads, key heads, queries, keys, extent), window, sinks
    ((1, 2, 1, 1, 70, 64), 0, 0),
    ((2, 4, 1, 1, 5003, 64), 0, 0),      # one token: keys in parts
    ((1, 1, 1, 1, 40000, 64), 0, 0),     # in many parts
    ((1, 3, 1, 1, 1, 40), 0, 0),         # one key
    ((1, 4, 2, 1, 300, 64), 1, 0),       # a window of one key
    ((1, 2, 1, 40, 2501, 64), 0, 0),     # workgroups of 16 rows, keys in parts
    ((4, 8, 8, 150, 1999, 32), 0, 0),    # tiles of rows, keys in parts
    ((8, 8, 4, 200, 200, 72), 50, 3),    # tiles of rows, window and sinks
    ((2, 2, 2, 330, 330, 128), 64, 20),
]
SIZES = {F32: (1e3, 1e4, 1e6, 1e9, 1e36), F64: (1e3, 1e9, 1e12, 1e19, 1e200)}


def signed_keys(shape, size, window, sinks, dtype, seed=21):
    """Inputs whose scores are size or -size (about, the same for all keys of a query):
    every key of a head is one vector or its opposite, every query lies along it.  With
    the exact weights: a query's visible keys of the larger score share them equally."""
    b, h, hk, t, s, d = shape
    rng = np.random.default_rng(seed)
    amplitude = np.sqrt(size / np.sqrt(d))
    one = rng.standard_normal((b, hk, 1, d))
    key_sign = np.where(rng.random((b, hk, s)) < 0.7, 1.0, -1.0)
    query_sign = np.where(rng.random((b, h, t)) < 0.5, 1.0, -1.0)
    along = np.repeat(one, h // hk, 1) * (1 + 0.1 * rng.random((b, h, t, d)))
    q = (amplitude * query_sign[..., None] * along).astype(dtype)
    k = (amplitude * key_sign[..., None] * one.astype(dtype)).astype(dtype)
    v, g = (rng.standard_normal(x).astype(dtype) for x in (k.shape, q.shape))
    seen = oracle.visible(t, s, [s] * b, window, sinks)[:, None]
    sign = np.where(seen, query_sign[..., None] * np.repeat(key_sign, h // hk, 1)[:, :, None],
                    -np.inf)
    top = sign.max(-1, keepdims=True)
    weight = ((sign == top) & seen).astype(F64)
    weight /= np.maximum(weight.sum(-1, keepdims=True), 1)
    return q, k, v, g, weight


@pytest.mark.parametrize("shape,window,sinks", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [F32, F64])
def test_equal_scores_have_equal_weights(hip, shape, window, sinks, dtype):
    """A weight before the division is 1 or 0 exactly, and their sum a whole number: what
    remains is the sum of values (a rounding a key), its parts, and the division."""
    b, h, hk, t, s, d = shape
    for size in SIZES[dtype]:
        q, k, v, _, weight = signed_keys(shape, size, window, sinks, dtype)
        output, _, _ = attend(hip, q, k, v, window, sinks, out_fill=7.0)
        values = np.repeat(v, h // hk, 1).astype(F64)
        assert_within(output, weight @ values,
                      (s + 40) * half_step(dtype) * (weight @ np.abs(values)), f"size {size}")
