"""Rotary positions, normed heads with the rotation, and windowed attention
against their definitions in 64 bits, through the C ABI."""
import ctypes

import numpy as np
import pytest

from tests import attention_oracle as oracle
from tests.attention_oracle import assert_within, half_step

pytestmark = pytest.mark.gpu

F32, F64 = np.float32, np.float64
_alive = []


@pytest.fixture(autouse=True)
def _release_buffers():
    yield
    _alive.clear()


class View:
    """A [batch, heads, tokens, extent] array in device memory: `order` "heads" (a
    head's tokens side by side) or "tokens" (a token's heads), the rows `gap`
    elements longer than a head's, and the first `offset` elements behind the
    buffer's start."""

    def __init__(self, hip, values, order="tokens", gap=0, offset=0, fill=0.0):
        b, h, t, d = values.shape
        self.hip, self.shape, self.dtype, self.order = hip, values.shape, values.dtype, order
        self.offset, self.pitch = offset, d + gap
        outer = (b, t, h) if order == "tokens" else (b, h, t)
        self.outer = outer
        whole = np.full(offset + b * h * t * self.pitch, fill, values.dtype)
        rows = whole[offset:].reshape(*outer, self.pitch)
        rows[..., :d] = values.transpose(0, 2, 1, 3) if order == "tokens" else values
        self.buffer = hip.DeviceBuffer.from_numpy(whole)
        self.count = whole.size
        _alive.append(self.buffer)
        steps = {"tokens": (t * h, 1, h), "heads": (h * t, t, 1)}[order]
        self.strides = tuple(s * self.pitch for s in steps)

    @property
    def heads(self):
        return self.hip.heads(self.buffer.address(self.offset * self.dtype.itemsize), self.strides)

    def numpy(self):
        whole = self.buffer.to_numpy(self.dtype, (self.count,))
        rows = whole[self.offset:].reshape(*self.outer, self.pitch)
        self.gaps = rows[..., self.shape[3]:]
        rows = rows[..., :self.shape[3]]
        return rows.transpose(0, 2, 1, 3) if self.order == "tokens" else rows


def device(hip, array):
    buffer = hip.DeviceBuffer.from_numpy(np.ascontiguousarray(array))
    _alive.append(buffer)
    return buffer


def space(hip, nbytes):
    buffer = hip.DeviceBuffer(max(int(nbytes), 16))
    _alive.append(buffer)
    return buffer


def tag(hip, dtype):
    return hip.dtype_tag(dtype)


# ------------------------------------------------------------------ rotation

ROTARY = [  # batch, heads, tokens, extent, rotary, layout, first position, dtype, magnitude
    (1, 1, 1, 2, 2, "half", 5, F32, 1.0),
    (2, 3, 7, 64, 64, "half", 0, F32, 1.0),
    (2, 3, 7, 64, 64, "interleaved", 0, F32, 1.0),
    (1, 5, 9, 80, 32, "interleaved", 131000, F32, 1.25),
    (3, 2, 5, 40, 22, "half", 1 << 20, F32, 0.5),
    (1, 4, 3, 33, 6, "half", 7, F32, 1.0),
    (2, 1, 4, 33, 10, "interleaved", 7, F32, 1.0),
    (1, 2, 3, 17, 0, "half", 7, F32, 2.0),
    (2, 3, 6, 256, 254, "half", 90000, F64, 1.0),
    (1, 3, 5, 30, 30, "interleaved", 1000, F64, 1.1),
    (1, 2, 3, 300, 298, "half", 1 << 29, F64, 1.0),
    (16, 17, 300, 64, 64, "half", 0, F32, 1.0),     # lanes that turn several heads
    (16, 9, 301, 128, 96, "interleaved", 3, F64, 1.0),
]


def rotary_of(hip, positions, freq, layout, magnitude, shared=False):
    positions = np.asarray(positions)
    return hip.rotary(device(hip, positions).ptr, 0 if shared else positions.shape[-1],
                      tag(hip, positions.dtype), device(hip, freq).ptr if len(freq) else None,
                      2 * len(freq), magnitude,
                      hip.ROTARY_HALF if layout == "half" else hip.ROTARY_INTERLEAVED)


@pytest.mark.parametrize("case", ROTARY, ids=str)
@pytest.mark.parametrize("inverse", [0, 1])
def test_rotary(hip, case, inverse):
    b, h, t, d, r, layout, start, dtype, magnitude = case
    rng = np.random.default_rng(7)
    x = rng.standard_normal((b, h, t, d)).astype(dtype)
    positions = start + 3 * np.arange(b)[:, None] + np.arange(t)
    freq = oracle.frequencies(r) if r else np.empty(0)
    source, target = View(hip, x, "tokens", gap=5, offset=1), View(hip, 0 * x, "heads", gap=3)
    hip.call("spar_hip_launch_rotary", target.heads, source.heads, b, h, t, d,
             rotary_of(hip, positions.astype(np.int32 if start % 2 else np.int64), freq, layout,
                       magnitude), inverse, tag(hip, dtype), 0)
    want, size = oracle.turn(x, positions, freq, layout, magnitude, bool(inverse))
    # angles of 2^29 turns: the product with the frequency is the same double in both
    assert_within(target.numpy(), want, oracle.TURN * half_step(dtype) * size)
    assert not target.gaps.any()


def test_rotary_in_place_shared_positions_and_far_angles(hip):
    rng = np.random.default_rng(8)
    x = rng.standard_normal((2, 3, 4, 64)).astype(F32)
    positions = np.array([0, -5, (1 << 31) + 12345, (1 << 40) + 7], np.int64)
    freq = oracle.frequencies(64)
    view = View(hip, x)
    hip.call("spar_hip_launch_rotary", view.heads, view.heads, 2, 3, 4, 64,
             rotary_of(hip, positions, freq, "half", 1.0, shared=True), 0, 0, 0)
    want, size = oracle.turn(x, positions, freq, "half")
    assert_within(view.numpy(), want, oracle.TURN * half_step(F32) * size)


# ------------------------------------------------------ head norm and rotation

NORMS = [  # batch, query heads, key heads, tokens, extent, rotary, layout, dtype
    (1, 1, 1, 1, 1, 0, "half", F32),
    (2, 4, 1, 3, 64, 64, "half", F32),
    (1, 3, 2, 5, 128, 128, "interleaved", F32),
    (2, 5, 5, 4, 72, 30, "half", F32),
    (1, 2, 1, 9, 100, 100, "half", F32),
    (3, 1, 2, 2, 33, 12, "interleaved", F32),
    (1, 6, 3, 4, 256, 254, "half", F64),
    (2, 2, 2, 3, 255, 64, "interleaved", F64),
    (4, 9, 3, 301, 64, 64, "half", F32),  # several heads per lane, every workgroup
    (3, 7, 2, 1001, 128, 64, "half", F64),
]


@pytest.mark.parametrize("case", NORMS, ids=str)
def test_head_norm_rotary(hip, case):
    b, hq, hk, t, d, r, layout, dtype = case
    rng = np.random.default_rng(9)
    # the packed projection: each token's query, key and value heads side by side
    packed = rng.standard_normal((b, hq + 2 * hk, t, d)).astype(dtype) * 2
    weights = [(1 + 0.3 * rng.standard_normal(d)).astype(dtype) for _ in range(2)]
    positions = 11 + np.arange(b)[:, None] * 5 + np.arange(t)
    freq = oracle.frequencies(r) if r else np.empty(0)
    source = View(hip, packed, "tokens", offset=1)
    heads = (hq, hk)
    begins = (0, hq)
    u = half_step(dtype)
    item = np.dtype(dtype).itemsize
    outputs = [View(hip, np.zeros((b, h, t, d), dtype), order)
               for h, order in zip(heads, ("tokens", "heads"))]
    saved = [space(hip, b * h * t * item) for h in heads]
    weight_buffers = [device(hip, w) for w in weights]
    inputs = [source.buffer.address((1 + at * d) * item) for at in begins]
    rotary = rotary_of(hip, positions, freq, layout, 1.1)
    parts = hip.head_norms(*(
        (out.heads.data, out.strides, s.ptr, x, source.strides, w.ptr, h)
        for out, s, x, w, h in zip(outputs, saved, inputs, weight_buffers, heads)))
    hip.call("spar_hip_launch_head_norm_rotary_forward", parts, 2, b, t, d, rotary, 1e-5,
             tag(hip, dtype), 0)
    slices = [packed[:, at:at + h] for at, h in zip(begins, heads)]
    for out, s, x, w, h in zip(outputs, saved, slices, weights, heads):
        y, size = oracle.norm(x, w.astype(F64), 1e-5)
        assert_within(s.to_numpy(dtype, (b, h, t)), size[..., 0], oracle.NORM * u * size[..., 0])
        want, scale = oracle.turn(y, positions, freq, layout, 1.1)
        assert_within(out.numpy(), want, (oracle.NORM + oracle.TURN) * u * scale)

    gradients = [rng.standard_normal((b, h, t, d)).astype(dtype) for h in heads]
    sources = [View(hip, g, order, gap=1) for g, order in zip(gradients, ("heads", "tokens"))]
    targets = [View(hip, np.zeros((b, h, t, d), dtype), order, gap=2)
               for h, order in zip(heads, ("tokens", "heads"))]
    weight_targets = [space(hip, d * item) for _ in heads]
    need = hip.head_norm_rotary_workspace(b, t, hq + hk, d, tag(hip, dtype))
    workspace = space(hip, need)
    parts = hip.head_norm_gradients(*(
        (dx.heads.data, dx.strides, dw.ptr, g.heads.data, g.strides, x, source.strides, w.ptr,
         s.ptr, h)
        for dx, dw, g, x, w, s, h in zip(targets, weight_targets, sources, inputs, weight_buffers,
                                         saved, heads)))
    hip.call("spar_hip_launch_head_norm_rotary_backward", parts, 2, b, t, d, rotary, workspace.ptr,
             need, tag(hip, dtype), 0)
    for dx, dw, g, x, w, h in zip(targets, weight_targets, gradients, slices, weights, heads):
        turned, size = oracle.turn(g, positions, freq, layout, 1.1, inverse=True)
        want, want_w, _, _ = oracle.norm_backward(x, w.astype(F64), turned, 1e-5)
        _, _, scale, scale_w = oracle.norm_backward(np.abs(x), np.abs(w.astype(F64)), size, 1e-5)
        # the turned gradient, d, and the mean's sum (9 additions), products and
        # the difference; dw's sum: at most 2 sqrt(rows) u beyond a tree's
        assert_within(dx.numpy(), want, (2 * oracle.NORM + oracle.TURN + 16) * u * scale)
        assert not dx.gaps.any()
        assert_within(dw.to_numpy(dtype, (d,)), want_w,
                      (oracle.NORM + oracle.TURN + 16 + 2 * np.sqrt(b * h * t)) * u * scale_w)


def test_head_norm_of_no_rows_has_no_weight_gradient(hip):
    d = 64
    dw = device(hip, np.full(d, 7.0, F32))
    rotary = hip.rotary(None, 0, hip.INT32, None, 0)
    parts = hip.head_norm_gradients((None, (0, 0, 0), dw.ptr, None, (0, 0, 0), None, (0, 0, 0),
                                     None, None, 4))
    hip.call("spar_hip_launch_head_norm_rotary_backward", parts, 1, 2, 0, d, rotary, None, 0, 0, 0)
    assert not dw.to_numpy(F32, (d,)).any()


# ----------------------------------------------------------------- attention

def attend(hip, q, k, v, window=0, sinks=0, scale=None, lengths=None, gradient=None,
           orders=("tokens", "tokens"), gap=0, offset=0, out_fill=0.0):
    """(output, logsumexp, gradients or None) of the C ABI."""
    dtype = q.dtype
    b, h, t, d = q.shape
    hk, s = k.shape[1:3]
    views = [View(hip, q, orders[0], gap, offset)] + [
        View(hip, x, orders[1], gap, offset) for x in (k, v)]
    length_buffer = None if lengths is None else device(hip, np.asarray(lengths))
    shape = hip.attention(b, h, hk, t, s, d, window, sinks,
                          1 / np.sqrt(d) if scale is None else scale,
                          None if lengths is None else length_buffer.ptr,
                          hip.INT32 if lengths is None else tag(hip, np.asarray(lengths).dtype),
                          tag(hip, dtype))
    out = View(hip, np.full(q.shape, out_fill, dtype), orders[0], gap, offset)
    saved = space(hip, b * h * t * dtype.itemsize)
    need = hip.attention_workspace(shape, 0)
    workspace = space(hip, need)
    hip.call("spar_hip_launch_attention_forward", out.heads, saved.ptr, *(x.heads for x in views),
             shape, workspace.ptr, need, 0)
    output, logsumexp = out.numpy(), saved.to_numpy(dtype, (b, h, t))
    assert not out.gaps.any()
    if gradient is None:
        return output, logsumexp, None
    need = hip.attention_workspace(shape, 1)
    workspace = space(hip, need)
    g = View(hip, gradient, orders[1], gap, offset)
    targets = [View(hip, np.full(x.shape, out_fill, dtype), order, gap, offset)
               for x, order in zip((q, k, v), (orders[0], orders[1], orders[1]))]
    hip.call("spar_hip_launch_attention_backward", *(x.heads for x in targets), g.heads, out.heads,
             saved.ptr, *(x.heads for x in views), shape, workspace.ptr, need, 0)
    made = [x.numpy() for x in targets]
    assert not any(x.gaps.any() for x in targets)
    return output, logsumexp, made


def inputs(b, h, hk, t, s, d, dtype, seed=3):
    rng = np.random.default_rng(seed)
    return [rng.standard_normal(shape).astype(dtype)
            for shape in ((b, h, t, d), (b, hk, s, d), (b, hk, s, d), (b, h, t, d))]


def check(hip, shape, dtype, window=0, sinks=0, lengths=None, **more):
    b, h, hk, t, s, d = shape
    q, k, v, g = inputs(*shape, dtype)
    want = oracle.Attention(q, k, v, window, sinks, more.get("scale"), lengths, dtype)
    output, logsumexp, made = attend(hip, q, k, v, window, sinks, lengths=lengths, gradient=g,
                                     out_fill=7.0, **more)
    assert_within(output, want.output, want.output_bound, "output")
    assert_within(logsumexp, want.logsumexp, want.logsumexp_bound, "logsumexp")
    gradients, bounds = want.backward(g)
    for name, x, y, bound in zip(("dq", "dk", "dv"), made, gradients, bounds):
        assert_within(x, y, bound, name)


ATTENTION = [  # (batch, heads, key heads, queries, keys, extent), window, sinks, lengths
    ((1, 1, 1, 1, 1, 1), 0, 0, None),
    ((2, 2, 1, 1, 5, 16), 0, 0, None),
    ((1, 4, 2, 3, 20, 33), 4, 2, None),
    ((2, 8, 8, 17, 17, 64), 0, 0, None),
    ((1, 6, 2, 65, 65, 64), 7, 3, None),
    ((2, 4, 1, 33, 70, 72), 16, 4, [70, 33]),
    ((3, 3, 3, 40, 40, 32), 9, 1, [40, 17, 0]),
    ((1, 2, 1, 130, 130, 100), 0, 5, None),
    ((1, 2, 2, 129, 200, 128), 1, 0, None),
    ((1, 2, 2, 97, 97, 96), 1, 1, None),
    ((1, 3, 1, 70, 70, 130), 33, 20, None),
    ((1, 2, 1, 64, 96, 192), 500, 4, None),
    ((1, 2, 1, 50, 81, 256), 20, 90, None),
    ((2, 2, 1, 9, 4, 40), 3, 1, [4, 1]),   # more queries than keys
    ((2, 2, 1, 5, 0, 40), 3, 1, None),     # no keys at all
    ((1, 8, 1, 300, 300, 64), 50, 70, None),  # sinks of two tiles, rows of one head group
    ((1, 5, 5, 256, 256, 3), 100, 0, None),
    ((1, 1, 1, 200, 200, 254), 64, 40, None),  # sinks that two waves share, odd pieces
    ((1, 7, 1, 90, 90, 64), 0, 0, None),       # a group that does not divide a tile of rows
    ((2, 3, 1, 400, 400, 48), 1000, 3, [400, 399]),  # a window that reaches over all keys
]


@pytest.mark.parametrize("shape,window,sinks,lengths", ATTENTION, ids=str)
@pytest.mark.parametrize("dtype", [F32, F64])
def test_attention(hip, shape, window, sinks, lengths, dtype):
    check(hip, shape, dtype, window, sinks, lengths)


def check_in_tiles(hip, shape, dtype, window=0, sinks=0, lengths=None, of_keys=False, **more):
    """The same shape for so many sequences that tiles of 64 rows (or `of_keys`) fill the
    chip, which then take them: the shape's sequences over and over, each repetition the
    same bits."""
    b, h, hk, t, s, d = shape
    times = -(-192 // (b * hk * -(-s // 64 if of_keys else -t * h // hk // 64)))
    q, k, v, g = inputs(*shape, dtype)
    want = oracle.Attention(q, k, v, window, sinks, more.get("scale"), lengths, dtype)
    lengths = None if lengths is None else np.tile(np.asarray(lengths), times)
    output, logsumexp, made = attend(hip, *(np.tile(x, (times, 1, 1, 1)) for x in (q, k, v)), window,
                                     sinks, lengths=lengths,
                                     gradient=np.tile(g, (times, 1, 1, 1)), out_fill=7.0, **more)
    for x in (output, logsumexp, *made):
        assert np.array_equal(x, np.tile(x[:b], (times,) + (1,) * (x.ndim - 1)))
    assert_within(output[:b], want.output, want.output_bound, "output")
    assert_within(logsumexp[:b], want.logsumexp, want.logsumexp_bound, "logsumexp")
    gradients, bounds = want.backward(g)
    for name, x, y, bound in zip(("dq", "dk", "dv"), made, gradients, bounds):
        assert_within(x[:b], y, bound, name)


@pytest.mark.parametrize("shape,window,sinks,lengths",
                         [case for case in ATTENTION if case[0][3] * case[0][1] // case[0][2] > 32],
                         ids=str)
@pytest.mark.parametrize("dtype", [F32, F64])
def test_attention_in_tiles(hip, shape, window, sinks, lengths, dtype):
    check_in_tiles(hip, shape, dtype, window, sinks, lengths)


@pytest.mark.parametrize("shape,window,sinks,lengths",
                         [case for case in ATTENTION if 16 <= case[0][4] <= 200], ids=str)
@pytest.mark.parametrize("dtype", [F32, F64])
def test_attention_in_tiles_of_keys(hip, shape, window, sinks, lengths, dtype):
    check_in_tiles(hip, shape, dtype, window, sinks, lengths, of_keys=True)


@pytest.mark.parametrize("shape,window,sinks,lengths", [
    ((1, 6, 6, 350, 350, 40), 330, 20, None),         # sinks of two tiles of 16 keys
    ((2, 8, 4, 250, 250, 72), 200, 3, [250, 101]),
    ((1, 5, 5, 333, 500, 66), 0, 0, None),
    ((1, 4, 2, 200, 1500, 64), 0, 0, None),           # and the keys of few rows
    ((2, 4, 2, 70, 1100, 40), 800, 5, [1100, 400]),
], ids=str)
@pytest.mark.parametrize("dtype", [F32, F64])
def test_work_of_small_grids_is_split(hip, shape, window, sinks, lengths, dtype):
    check(hip, shape, dtype, window, sinks, lengths)


@pytest.mark.parametrize("orders,gap,offset", [(("heads", "heads"), 4, 4),
                                               (("tokens", "heads"), 3, 1)])
@pytest.mark.parametrize("extent", [64, 66])
def test_attention_layouts_in_tiles(hip, orders, gap, offset, extent):
    check_in_tiles(hip, (2, 6, 2, 80, 90, extent), F32, 21, 3, np.array([90, 61], np.int64),
                   orders=orders, gap=gap, offset=offset, scale=0.3)


@pytest.mark.parametrize("orders,gap,offset", [(("heads", "heads"), 0, 0),
                                               (("tokens", "heads"), 3, 1),
                                               (("heads", "tokens"), 1, 3)])
@pytest.mark.parametrize("queries", [2, 80])
def test_attention_layouts(hip, orders, gap, offset, queries):
    check(hip, (2, 4, 2, queries, 90, 66), F32, 21, 3, np.array([90, 61], np.int64), orders=orders,
          gap=gap, offset=offset, scale=0.3)


@pytest.mark.parametrize("shape,window,sinks,lengths", [
    ((2, 4, 1, 1, 5003, 64), 0, 0, [5003, 1700]),      # keys split, four rows
    ((1, 16, 1, 2, 4001, 128), 3000, 4, None),          # two tiles of rows
    ((1, 2, 1, 40, 2501, 64), 0, 0, None),              # tiles of rows, keys split
    ((2, 4, 4, 150, 1999, 80), 900, 7, [1999, 3]),
], ids=str)
@pytest.mark.parametrize("dtype", [F32, F64])
def test_attention_of_split_keys(hip, shape, window, sinks, lengths, dtype):
    check(hip, shape, dtype, window, sinks, lengths)


def test_attention_fills_the_grid_with_two_blocks_of_rows(hip):
    check(hip, (16, 8, 8, 520, 520, 64), F32, 130, 4)


def test_sinks_of_many_later_rows_are_split(hip):
    check(hip, (1, 4, 1, 2100, 2100, 32), F32, 8, 4)


def test_empty_rows_are_zero_and_give_no_gradient(hip):
    """Queries of empty or short sequences, with NaN in what they hold."""
    q, k, v, g = inputs(2, 2, 1, 6, 8, 64, F32)
    lengths = np.array([0, 4], np.int32)
    q[0] = g[0] = np.nan
    q[1, :, :2] = g[1, :, :2] = np.nan
    output, logsumexp, (dq, dk, dv) = attend(hip, q, k, v, 3, 1, lengths=lengths, gradient=g,
                                             out_fill=7.0)
    want = oracle.Attention(q, k, v, 3, 1, None, lengths)
    assert not output[0].any() and not output[1, :, :2].any()
    assert np.isneginf(logsumexp[0]).all() and np.isneginf(logsumexp[1, :, :2]).all()
    assert not dq[0].any() and not dq[1, :, :2].any() and not dk[0].any() and not dv[0].any()
    assert_within(output, want.output, want.output_bound)
    for x, y, bound in zip((dq, dk, dv), *want.backward(g)):
        assert_within(x, y, bound)


@pytest.mark.parametrize("queries", [1, 2, 70])
@pytest.mark.parametrize("garbage", [np.nan, np.inf, -np.inf, np.finfo(F32).max,
                                     -np.finfo(F32).max])
def test_what_no_query_sees_has_no_part(hip, queries, garbage):
    """Keys behind a sequence's length, and between its sinks and its window."""
    s, window, sinks = 300, 40, 3
    q, k, v, g = inputs(2, 4, 2, queries, s, 64, F32)
    lengths = np.array([s, 211], np.int32)
    for b, n in enumerate(lengths):
        for x in (k, v):
            x[b, :, n:] = garbage
            x[b, :, sinks:n - queries - window + 1] = garbage
    output, logsumexp, made = attend(hip, q, k, v, window, sinks, lengths=lengths, gradient=g)
    want = oracle.Attention(q, k, v, window, sinks, None, lengths)
    assert_within(output, want.output, want.output_bound)
    for x, y, bound in zip(made, *want.backward(g)):
        assert_within(x, y, bound)


def test_scores_of_the_lowest_value_and_large_scores(hip):
    """Scores near float32's ends stay finite in the softmax."""
    q, k, v, g = inputs(1, 2, 1, 20, 20, 32, F32)
    q *= 1e18
    k *= 1e18
    output, _, _ = attend(hip, q, k, v)
    want = oracle.Attention(q, k, v)
    # one key takes all the weight of a row: the scores differ by far more than 1
    assert_within(output, want.output, 1e-3 * np.abs(want.output) + 1e-6)


def test_a_nan_stays_in_its_sequence_and_head_group(hip):
    q, k, v, g = inputs(2, 4, 2, 40, 40, 64, F32)
    clean, _, _ = attend(hip, q, k, v, 10, 2)
    k[1, 1, 20] = np.nan
    q[0, 0, 5] = np.nan
    output, _, _ = attend(hip, q, k, v, 10, 2)
    assert np.isnan(output[0, 0, 5]).all() and np.isnan(output[1, 2:, 20:30]).all()
    assert np.array_equal(output[0, 1:], clean[0, 1:]) and np.array_equal(output[1, :2], clean[1, :2])
    assert np.array_equal(np.delete(output[0, 0], 5, 0), np.delete(clean[0, 0], 5, 0))


@pytest.mark.parametrize("shape", [(2, 4, 2, 1, 3001, 64), (1, 4, 1, 300, 300, 64)])
def test_results_do_not_change_from_run_to_run(hip, shape):
    q, k, v, g = inputs(*shape, F32)
    runs = [attend(hip, q, k, v, 100, 4, gradient=g) for _ in range(2)]
    assert np.array_equal(runs[0][0], runs[1][0]) and np.array_equal(runs[0][1], runs[1][1])
    for x, y in zip(runs[0][2], runs[1][2]):
        assert np.array_equal(x, y)


def test_gradients_against_differences(hip):
    """dL of L = sum(output * g) along random directions, in double: central
    differences of step 1e-4 are off by the third derivative times 1e-8 / 6."""
    q, k, v, g = inputs(2, 4, 2, 19, 23, 24, F64)
    args = dict(window=6, sinks=2, lengths=np.array([23, 20], np.int32))
    _, _, made = attend(hip, q, k, v, gradient=g, **args)
    rng = np.random.default_rng(4)
    for i in range(3):
        direction = rng.standard_normal((q, k, v)[i].shape)
        sides = []
        for step in (1e-4, -1e-4):
            moved = [x + step * direction if j == i else x for j, x in enumerate((q, k, v))]
            sides.append(np.sum(attend(hip, *moved, **args)[0] * g))
        difference = (sides[0] - sides[1]) / 2e-4
        along = np.sum(made[i] * direction)
        assert abs(difference - along) <= 1e-6 * np.sum(np.abs(made[i] * direction)), i


def test_cache_offsets_beyond_32_bits(hip):
    """One sequence of 2 key heads whose second head begins 2^32 + elements behind
    the first: byte and element offsets pass 32 bits."""
    d, s = 64, 400
    step = (1 << 32) + 4096
    q, k, v, _ = inputs(1, 2, 2, 1, s, d, F32)
    buffers = []
    for x in (k, v):
        buffer = space(hip, (step + s * d) * 4)
        for head in range(2):
            part = np.ascontiguousarray(x[0, head])
            hip.call("spar_hip_copy_host_to_device", buffer.address(head * step * 4),
                     part.ctypes.data, part.nbytes, 0)
        buffers.append(hip.heads(buffer.ptr, (0, step, d)))
    shape = hip.attention(1, 2, 2, 1, s, d, 0, 0, 0.125, None, hip.INT32, 0)
    need = hip.attention_workspace(shape, 0)
    query, out = View(hip, q), View(hip, 0 * q)
    hip.call("spar_hip_launch_attention_forward", out.heads, None, query.heads, *buffers, shape,
             space(hip, need).ptr, need, 0)
    want = oracle.Attention(q, k, v)
    assert_within(out.numpy(), want.output, want.output_bound)
    _alive.clear()
    hip.call("spar_hip_empty_cache", 0)


def test_rotary_offsets_beyond_32_bits(hip):
    """Two heads 2^32 + 4096 elements apart, turned in place."""
    d, t = 64, 5
    step = (1 << 32) + 4096
    x = np.random.default_rng(6).standard_normal((1, 2, t, d)).astype(F32)
    buffer = space(hip, (step + t * d) * 4)
    for head in range(2):
        part = np.ascontiguousarray(x[0, head])
        hip.call("spar_hip_copy_host_to_device", buffer.address(head * step * 4),
                 part.ctypes.data, part.nbytes, 0)
    view = hip.heads(buffer.ptr, (0, step, d))
    freq = oracle.frequencies(d)
    hip.call("spar_hip_launch_rotary", view, view, 1, 2, t, d,
             rotary_of(hip, np.arange(t), freq, "half", 1.0, shared=True), 0, 0, 0)
    want, size = oracle.turn(x, np.arange(t), freq, "half")
    for head in range(2):
        got = np.empty((t, d), F32)
        hip.call("spar_hip_copy_device_to_host", got.ctypes.data, buffer.address(head * step * 4),
                 got.nbytes, 0)
        assert_within(got, want[0, head], oracle.TURN * half_step(F32) * size[0, head])
    _alive.clear()
    hip.call("spar_hip_empty_cache", 0)


# ------------------------------------------------------- a captured graph

def runtime():
    return ctypes.CDLL("libamdhip64.so")


def test_captured_runs_repeat_with_new_inputs(hip):
    """Norm and rotation, attention and both gradients recorded into a graph on the
    backend's stream: every replay gives what eager calls give for what the buffers
    hold then, with eager work in between."""
    b, h, hk, t, d = 2, 4, 2, 96, 64
    rng = np.random.default_rng(5)
    freq = device(hip, oracle.frequencies(d))
    positions = device(hip, np.arange(t, dtype=np.int64))
    rotary = hip.rotary(positions.ptr, 0, hip.INT64, freq.ptr, d)
    weight = device(hip, np.ones(d, F32))
    zeros = [np.zeros((b, n, t, d), F32) for n in (h, hk, hk, h)]
    x, v, g = View(hip, zeros[0]), View(hip, zeros[2]), View(hip, zeros[3])
    kx = View(hip, zeros[1])
    lengths = device(hip, np.array([t, t], np.int32))
    shape = hip.attention(b, h, hk, t, t, d, 30, 2, 0.125, lengths.ptr, hip.INT32, 0)

    def buffers():
        made = {n: View(hip, zeros[0]) for n in ("q", "out", "dq", "dx")}
        made |= {n: View(hip, zeros[1]) for n in ("k", "dk", "dv", "dkx")}
        made["rows"] = space(hip, b * (h + hk) * t * 4)
        made["lse"] = space(hip, b * h * t * 4)
        made["dw"] = space(hip, 2 * d * 4)
        needs = [hip.attention_workspace(shape, 0), hip.attention_workspace(shape, 1),
                 hip.head_norm_rotary_workspace(b, t, h + hk, d, 0)]
        made["work"] = [(space(hip, n), n) for n in needs]
        return made

    def run(m):
        split = m["rows"].ptr + b * h * t * 4
        hip.call("spar_hip_launch_head_norm_rotary_forward", hip.head_norms(
            (m["q"].heads.data, m["q"].strides, m["rows"].ptr, x.heads.data, x.strides, weight.ptr,
             h),
            (m["k"].heads.data, m["k"].strides, split, kx.heads.data, kx.strides, weight.ptr, hk)),
            2, b, t, d, rotary, 1e-5, 0, 0)
        (w0, n0), (w1, n1), (w2, n2) = m["work"]
        hip.call("spar_hip_launch_attention_forward", m["out"].heads, m["lse"].ptr, m["q"].heads,
                 m["k"].heads, v.heads, shape, w0.ptr, n0, 0)
        hip.call("spar_hip_launch_attention_backward", m["dq"].heads, m["dk"].heads, m["dv"].heads,
                 g.heads, m["out"].heads, m["lse"].ptr, m["q"].heads, m["k"].heads, v.heads, shape,
                 w1.ptr, n1, 0)
        hip.call("spar_hip_launch_head_norm_rotary_backward", hip.head_norm_gradients(
            (m["dx"].heads.data, m["dx"].strides, m["dw"].ptr, m["dq"].heads.data, m["dq"].strides,
             x.heads.data, x.strides, weight.ptr, m["rows"].ptr, h),
            (m["dkx"].heads.data, m["dkx"].strides, m["dw"].ptr + d * 4, m["dk"].heads.data,
             m["dk"].strides, kx.heads.data, kx.strides, weight.ptr, split, hk)),
            2, b, t, d, rotary, w2.ptr, n2, 0, 0)

    def refill(seed, newest):
        rng = np.random.default_rng(seed)
        for view in (x, kx, v, g):
            values = rng.standard_normal(view.count).astype(F32)
            hip.call("spar_hip_copy_host_to_device", view.buffer.ptr, values.ctypes.data,
                     values.nbytes, 0)
        values = np.array([t, newest], np.int32)
        hip.call("spar_hip_copy_host_to_device", lengths.ptr, values.ctypes.data, 8, 0)

    captured, eager = buffers(), buffers()
    refill(0, t)
    run(captured)  # first use of every kernel outside the capture
    hip.synchronize()
    lib = runtime()
    stream, graph, executable = (ctypes.c_void_p() for _ in range(3))
    hip.call("spar_hip_stream", ctypes.byref(stream), 0)
    assert lib.hipStreamBeginCapture(stream, 2) == 0
    run(captured)
    assert lib.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert lib.hipGraphInstantiate(ctypes.byref(executable), graph, None, None, 0) == 0
    names = ("q", "k", "out", "dq", "dk", "dv", "dx", "dkx")
    for seed, newest in ((1, t), (2, 50), (3, 0), (4, 1)):
        refill(seed, newest)
        run(eager)
        assert lib.hipGraphLaunch(executable, stream) == 0
        hip.synchronize()
        for name in names:
            assert np.array_equal(captured[name].numpy(), eager[name].numpy()), (seed, name)
        assert np.array_equal(captured["dw"].to_numpy(F32, (2 * d,)),
                              eager["dw"].to_numpy(F32, (2 * d,)))
    lib.hipGraphExecDestroy(executable)
    lib.hipGraphDestroy(graph)
