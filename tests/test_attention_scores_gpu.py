"""Attention of keys whose scores are equal or opposite: the exact weights are known at
any size of score, so that what a score's rounding costs is not part of the bounds."""
import numpy as np
import pytest

from tests import attention_oracle as oracle
from tests.attention_oracle import assert_within, half_step
from tests.test_attention_gpu import F32, F64, _release_buffers, attend, inputs  # noqa: F401

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
    """A query's weights before the division are one number or 0 exactly.  What remains is
    the sum of weights and that of values (a rounding a key each), their parts, and the
    division."""
    b, h, hk, t, s, d = shape
    for size in SIZES[dtype]:
        q, k, v, _, weight = signed_keys(shape, size, window, sinks, dtype)
        output, _, _ = attend(hip, q, k, v, window, sinks, out_fill=7.0)
        values = np.repeat(v, h // hk, 1).astype(F64)
        assert_within(output, weight @ values,
                      (2 * s + 40) * half_step(dtype) * (weight @ np.abs(values)), f"size {size}")


@pytest.mark.parametrize("shape,window,sinks", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [F32, F64])
def test_gradients_of_equal_scores(hip, shape, window, sinks, dtype):
    """Weights as above, off by the sum of weights (a rounding a key) and the division."""
    b, h, hk, t, s, d = shape
    group, u, scale = h // hk, half_step(dtype), 1 / np.sqrt(d)

    def over_groups(x):
        return x.reshape(b, hk, group, *x.shape[2:]).sum(2)

    for size in SIZES[dtype]:
        q, k, v, g, weight = signed_keys(shape, size, window, sinks, dtype)
        _, _, (dq, dk, dv) = attend(hip, q, k, v, window, sinks, gradient=g, out_fill=7.0)
        q, g = q.astype(F64), g.astype(F64)
        k, v = (np.repeat(x, group, 1).astype(F64) for x in (k, v))
        weight_t = weight.swapaxes(2, 3)
        output = weight @ v
        ds = weight * (g @ v.swapaxes(2, 3) - (g * output).sum(-1, keepdims=True))
        ds_t = ds.swapaxes(2, 3)
        # dP and delta: products of d numbers and their sums, and the output's own error
        size_of = np.abs(g) @ np.abs(v).swapaxes(2, 3) + (
            np.abs(g) * (weight @ np.abs(v))).sum(-1, keepdims=True)
        ds_bound = weight * u * (d + 3 * s + 60) * size_of
        rows = t * group + 80
        assert_within(dq, scale * (ds @ k), scale * (
            ds_bound @ np.abs(k) + u * (s + 40) * (np.abs(ds) @ np.abs(k))), f"dq {size}")
        assert_within(dk, scale * over_groups(ds_t @ q), scale * over_groups(
            ds_bound.swapaxes(2, 3) @ np.abs(q) + u * rows * (np.abs(ds_t) @ np.abs(q))),
            f"dk {size}")
        assert_within(dv, over_groups(weight_t @ g),
                      u * (s + 10 + rows) * over_groups(weight_t @ np.abs(g)), f"dv {size}")


@pytest.mark.parametrize("scale", [0.0, -0.7, 1e-30, 8.0 / np.log2(np.e), 3.3])
@pytest.mark.parametrize("shape,window,sinks", [((1, 2, 1, 9, 70, 40), 0, 0),
                                                ((8, 8, 4, 200, 200, 64), 50, 3)], ids=str)
@pytest.mark.parametrize("dtype", [F32, F64])
def test_scales(hip, shape, window, sinks, scale, dtype):
    """Scales of any sign and size, whose powers of two the backward takes apart.  Weights
    below the smallest normal number may be zero, which adds `tiny` to a weight's bound:
    the exponential of float32 rounds them so."""
    b, h, hk, t, keys, d = shape
    q, k, v, g = inputs(*shape, dtype)
    want = oracle.Attention(q, k, v, window, sinks, scale, None, dtype)
    output, logsumexp, made = attend(hip, q, k, v, window, sinks, scale, gradient=g, out_fill=7.0)
    tiny = np.finfo(dtype).tiny * want.seen
    assert_within(output, want.output, want.output_bound + tiny @ np.abs(want.v), "output")
    assert_within(logsumexp, want.logsumexp, want.logsumexp_bound, "logsumexp")
    gradients, bounds = want.backward(g)
    g = g.astype(F64)
    ds = tiny * np.abs(g @ want.v.swapaxes(2, 3) - (g * want.output).sum(-1, keepdims=True))

    def over_groups(x):
        return x.reshape(b, hk, h // hk, keys, d).sum(2)

    more = (abs(scale) * (ds @ np.abs(want.k)),
            abs(scale) * over_groups(ds.swapaxes(2, 3) @ np.abs(want.q)),
            over_groups(tiny.swapaxes(2, 3) @ np.abs(g)))
    for name, x, y, bound, flushed in zip(("dq", "dk", "dv"), made, gradients, bounds, more):
        assert_within(x, y, bound + flushed, name)
