"""Head norms with the rotation on their own inputs, and of one tensor, through the C ABI."""
import numpy as np
import pytest

from tests import attention_oracle as oracle
from tests.attention_oracle import assert_within, half_step
from tests.test_attention_gpu import _release_buffers  # noqa: F401
from tests.test_attention_gpu import F32, F64, View, device, rotary_of, space, tag

pytestmark = pytest.mark.gpu

SHAPES = [  # batch, heads of each part, tokens, extent
    (2, (5,), 3, 64),
    (1, (3, 2), 7, 40),
    # lanes that take several heads of a token, the last fewer than the others
    (4, (9, 3), 1100, 64),
    (4, (5,), 2500, 72),
    (2, (7, 1), 3300, 64),
]


def case(hip, shape, dtype, layout):
    b, heads, t, d = shape
    rng = np.random.default_rng(41)
    positions = 3 + np.arange(b)[:, None] + np.arange(t)
    freq = oracle.frequencies(32)
    xs = [rng.standard_normal((b, h, t, d)).astype(dtype) for h in heads]
    weights = [(1 + 0.3 * rng.standard_normal(d)).astype(dtype) for _ in heads]
    gradients = [rng.standard_normal(x.shape).astype(dtype) for x in xs]
    return xs, weights, gradients, positions, freq, rotary_of(hip, positions, freq, layout, 1.1)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [F32, F64])
def test_head_norms_on_their_own_inputs(hip, shape, layout, dtype):
    b, heads, t, d = shape
    u, item = half_step(dtype), np.dtype(dtype).itemsize
    xs, weights, gradients, positions, freq, rotary = case(hip, shape, dtype, layout)
    sources = [View(hip, x, order, gap=3) for x, order in zip(xs, ("tokens", "heads"))]
    kept = [View(hip, x) for x in xs]
    saved = [space(hip, b * h * t * item) for h in heads]
    weight_buffers = [device(hip, w) for w in weights]
    parts = hip.head_norms(*((x.heads.data, x.strides, s.ptr, x.heads.data, x.strides, w.ptr, h)
                             for x, s, w, h in zip(sources, saved, weight_buffers, heads)))
    hip.call("spar_hip_launch_head_norm_rotary_forward", parts, len(heads), b, t, d, rotary, 1e-5,
             tag(hip, dtype), 0)
    for x, view, s, w, h in zip(xs, sources, saved, weights, heads):
        y, size = oracle.norm(x, w.astype(F64), 1e-5)
        want, scale = oracle.turn(y, positions, freq, layout, 1.1)
        assert_within(view.numpy(), want, (oracle.NORM + oracle.TURN) * u * scale)
        assert not view.gaps.any()
        assert_within(s.to_numpy(dtype, (b, h, t)), size[..., 0], oracle.NORM * u * size[..., 0])

    targets = [View(hip, g, order, gap=1) for g, order in zip(gradients, ("heads", "tokens"))]
    weight_targets = [space(hip, d * item) for _ in heads]
    need = hip.head_norm_rotary_workspace(b, t, sum(heads), d, tag(hip, dtype))
    parts = hip.head_norm_gradients(*(
        (g.heads.data, g.strides, dw.ptr, g.heads.data, g.strides, x.heads.data, x.strides, w.ptr,
         s.ptr, h)
        for g, dw, x, w, s, h in zip(targets, weight_targets, kept, weight_buffers, saved, heads)))
    hip.call("spar_hip_launch_head_norm_rotary_backward", parts, len(heads), b, t, d, rotary,
             space(hip, need).ptr, need, tag(hip, dtype), 0)
    for view, dw, g, x, w, h in zip(targets, weight_targets, gradients, xs, weights, heads):
        w = w.astype(F64)
        turned, size = oracle.turn(g, positions, freq, layout, 1.1, inverse=True)
        want, want_w, _, _ = oracle.norm_backward(x, w, turned, 1e-5)
        _, _, scale, scale_w = oracle.norm_backward(np.abs(x), np.abs(w), size, 1e-5)
        # counted as for separate outputs: the turned gradient, d, the mean's sum, products
        # and the difference; dw's sum at most 2 sqrt(rows) u beyond a tree's
        assert_within(view.numpy(), want, (2 * oracle.NORM + oracle.TURN + 16) * u * scale)
        assert not view.gaps.any()
        assert_within(dw.to_numpy(dtype, (d,)), want_w,
                      (oracle.NORM + oracle.TURN + 16 + 2 * np.sqrt(b * h * t)) * u * scale_w)
