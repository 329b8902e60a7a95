"""The attention operators through the tensor API: a decoder layer's run from the
packed projection to the merged heads, views, gradients and refusals."""
import numpy as np
import pytest
import torch

from tests import attention_oracle as oracle
from tests.attention_oracle import assert_within

pytestmark = pytest.mark.gpu

F32, F64 = np.float32, np.float64


@pytest.fixture(scope="module")
def sp():
    from spar_amd import spar

    if spar.hip_device_count() < 1:
        pytest.fail("no HIP device visible to a gpu-marked test")
    return spar


def put(sp, array, grad=False):
    tensor = sp.Tensor.from_numpy(np.ascontiguousarray(array)).to(sp.Device.hip(0))
    if grad:
        tensor.set_requires_grad(True)
    return tensor


def get(sp, tensor):
    return tensor.contiguous().to(sp.Device.cpu()).numpy()


def layer(sp, packed, query_weight, key_weight, positions, freq, heads, key_heads, window, sinks,
          lengths, layout):
    """[batch, tokens, heads * extent] of the packed [batch, tokens, (q, k, v) heads *
    extent] projection: how a decoder layer uses the operators together."""
    b, t, width = packed.shape
    d = width // (heads + 2 * key_heads)
    every = packed.reshape([b, t, heads + 2 * key_heads, d]).transpose(1, 2)
    query, key = sp.query_key_norm_rotary(
        every.narrow(1, 0, heads), every.narrow(1, heads, key_heads), query_weight, key_weight,
        positions, freq, layout)
    value = every.narrow(1, heads + key_heads, key_heads)
    out = sp.window_attention(query, key, value, window, sinks, lengths=lengths)
    return out.transpose(1, 2).reshape([b, t, heads * d])


def layer_in_torch(packed, query_weight, key_weight, positions, freq, heads, key_heads, window,
                   sinks, lengths, layout):
    b, t, width = packed.shape
    d = width // (heads + 2 * key_heads)
    every = packed.reshape(b, t, heads + 2 * key_heads, d).transpose(1, 2)
    angle = torch.tensor(positions, dtype=torch.float64)[:, None] * torch.tensor(freq)
    cos, sin = angle.cos(), angle.sin()
    a, c = (torch.tensor(x) for x in oracle.pairs(2 * len(freq), layout))

    def normed(x, weight):
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * weight
        turned = y.clone()
        turned[..., a] = y[..., a] * cos - y[..., c] * sin
        turned[..., c] = y[..., c] * cos + y[..., a] * sin
        return turned

    q = normed(every[:, :heads], query_weight)
    k = normed(every[:, heads:heads + key_heads], key_weight)
    v = every[:, heads + key_heads:]
    k, v = (x.repeat_interleave(heads // key_heads, 1) for x in (k, v))
    seen = torch.tensor(oracle.visible(t, t, lengths, window, sinks))[:, None]
    scores = torch.where(seen, q @ k.transpose(2, 3) / d ** 0.5,
                         torch.tensor(-1e300, dtype=torch.float64))
    out = (torch.softmax(scores, -1) * seen) @ v
    return out.transpose(1, 2).reshape(b, t, heads * d)


@pytest.mark.parametrize("shape,window,sinks,lengths,rotary,layout", [
    ((2, 37, 4, 2, 64), 9, 2, [37, 20], 64, "half"),
    ((1, 130, 6, 1, 40), 50, 0, [130], 22, "interleaved"),
    ((3, 5, 2, 2, 8), 0, 0, [5, 0, 1], 8, "half"),
])
def test_decoder_layer(sp, shape, window, sinks, lengths, rotary, layout):
    """In double.  Norms, rotation and attention round a value a few hundred times in
    all (u = 1.1e-16, scores up to about 16 in size, so weights to some thousand u);
    1e-11 of the largest value leaves each gradient 10^5 u."""
    b, t, h, hk, d = shape
    rng = np.random.default_rng(12)
    arrays = [rng.standard_normal((b, t, (h + 2 * hk) * d)), 1 + 0.3 * rng.standard_normal(d),
              1 + 0.3 * rng.standard_normal(d)]
    g = rng.standard_normal((b, t, h * d))
    freq, positions = oracle.frequencies(rotary), 100 + np.arange(t)
    leaves = [torch.tensor(x, requires_grad=True) for x in arrays]
    want = layer_in_torch(*leaves, positions, freq, h, hk, window, sinks, lengths, layout)
    want.backward(torch.tensor(g))
    tensors = [put(sp, x, grad=True) for x in arrays]
    got = layer(sp, *tensors, put(sp, positions), put(sp, freq), h, hk, window, sinks,
                put(sp, np.array(lengths)),
                sp.RotaryLayout.Half if layout == "half" else sp.RotaryLayout.Interleaved)
    sp.sum(sp.multiply(got, put(sp, g))).backward()
    for x, y in [(get(sp, got), want)] + [(get(sp, s.grad()), l.grad)
                                          for s, l in zip(tensors, leaves)]:
        y = y.detach().numpy()
        assert np.max(np.abs(x - y)) <= 1e-11 * np.max(np.abs(y))


@pytest.mark.parametrize("kind", ["narrowed", "expanded", "columns"])
def test_rotary_of_views(sp, kind):
    rng = np.random.default_rng(13)
    x = rng.standard_normal((2, 5, 7, 12)).astype(F32)
    freq, positions = oracle.frequencies(6), np.arange(7, dtype=np.int32)
    if kind == "narrowed":
        leaf = put(sp, x, grad=True)
        view, values = leaf.narrow(3, 2, 8).narrow(2, 1, 5), x[:, :, 1:6, 2:10]
    elif kind == "expanded":
        leaf = put(sp, x[:, :1], grad=True)
        view, values = leaf.expand([2, 5, 7, 12]), np.broadcast_to(x[:, :1], x.shape)
    else:
        leaf = put(sp, x, grad=True)
        view, values = leaf.transpose(2, 3), x.swapaxes(2, 3)
        positions = np.arange(12, dtype=np.int32)
    positions = positions[:values.shape[2]]
    out = sp.rotary_embedding(view, put(sp, positions), put(sp, freq))
    want, size = oracle.turn(values, positions, freq, "half")
    bound = oracle.TURN * oracle.half_step(F32)
    assert_within(get(sp, out), want, bound * size)
    g = rng.standard_normal(values.shape).astype(F32)
    sp.sum(sp.multiply(out, put(sp, g))).backward()
    turned, size = oracle.turn(g, positions, freq, "half", inverse=True)
    if kind == "narrowed":
        want, scale = np.zeros(x.shape), np.zeros(x.shape)
        want[:, :, 1:6, 2:10], scale[:, :, 1:6, 2:10] = turned, size
    elif kind == "expanded":  # a sum of five: four roundings
        want, scale = (y.sum(1, keepdims=True) for y in (turned, 1.5 * size))
    else:
        want, scale = turned.swapaxes(2, 3), size.swapaxes(2, 3)
    assert_within(get(sp, leaf.grad()), want, bound * scale)


def test_outputs_lie_as_their_inputs(sp):
    x = np.zeros((2, 9, 4, 16), F32)
    tokens = put(sp, x).transpose(1, 2)  # a token's heads side by side
    heads = put(sp, x.transpose(0, 2, 1, 3))
    freq, positions = put(sp, oracle.frequencies(16)), put(sp, np.arange(9))
    weight = put(sp, np.ones(16, F32))
    for view, is_tokens in ((tokens, True), (heads, False)):
        outs = [sp.rotary_embedding(view, positions, freq), sp.window_attention(view, view, view),
                *sp.query_key_norm_rotary(view, view, weight, weight, positions, freq)]
        for out in outs:
            assert list(out.shape) == [2, 4, 9, 16]
            assert (out.transpose(1, 2) if is_tokens else out).is_contiguous()


@pytest.mark.parametrize("tracked", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)])
def test_some_inputs_tracked(sp, tracked):
    rng = np.random.default_rng(14)
    arrays = [rng.standard_normal(s).astype(F32) for s in ((1, 4, 6, 32), (1, 2, 9, 32),
                                                          (1, 2, 9, 32))]
    g = rng.standard_normal((1, 4, 6, 32)).astype(F32)
    tensors = [put(sp, x, grad=bool(t)) for x, t in zip(arrays, tracked)]
    out = sp.window_attention(*tensors, 4, 1, scale=0.2)
    sp.sum(sp.multiply(out, put(sp, g))).backward()
    want = oracle.Attention(*arrays, 4, 1, 0.2)
    assert_within(get(sp, out), want.output, want.output_bound)
    for tensor, track, value, bound in zip(tensors, tracked, *want.backward(g)):
        assert tensor.has_grad == bool(track)
        if track:
            assert_within(get(sp, tensor.grad()), value, bound)


def test_one_tensor_as_query_key_and_value(sp):
    """The gradients of a tensor used three times add up."""
    rng = np.random.default_rng(15)
    x = rng.standard_normal((2, 2, 11, 20))
    g = rng.standard_normal(x.shape)
    leaf = put(sp, x, grad=True)
    sp.sum(sp.multiply(sp.window_attention(leaf, leaf, leaf, 5, 1), put(sp, g))).backward()
    want = oracle.Attention(x, x, x, 5, 1, dtype=F64)
    gradients, bounds = want.backward(g)
    total = sum(gradients)
    assert_within(get(sp, leaf.grad()), total, sum(bounds) + 1e-15 * np.abs(total))


@pytest.mark.parametrize("shape", [(0, 2, 3, 8), (2, 2, 0, 8)])
def test_nothing(sp, shape):
    x = put(sp, np.zeros(shape, F32), grad=True)
    weight = put(sp, np.ones(8, F32))
    positions, freq = put(sp, np.arange(shape[2])), put(sp, oracle.frequencies(8))
    assert list(sp.rotary_embedding(x, positions, freq).shape) == list(shape)
    assert list(sp.window_attention(x, x, x).shape) == list(shape)
    query, key = sp.query_key_norm_rotary(x, x, weight, weight, positions, freq)
    assert list(query.shape) == list(key.shape) == list(shape)


def test_refusals(sp):
    x = put(sp, np.zeros((2, 4, 3, 8), F32))
    wide = put(sp, np.zeros((1, 1, 1, 258), F32))
    weight = put(sp, np.ones(8, F32))
    positions, freq = put(sp, np.arange(3)), put(sp, oracle.frequencies(8))
    three = put(sp, np.zeros((2, 3, 3, 8), F32))
    double = put(sp, np.zeros((2, 4, 3, 8)))
    turn, norm, attend = sp.rotary_embedding, sp.query_key_norm_rotary, sp.window_attention
    nan = float("nan")
    for call in (
            lambda: turn(x, put(sp, np.arange(4)), freq),
            lambda: turn(x, put(sp, np.zeros((3, 3), np.int64)), freq),
            lambda: turn(x, put(sp, np.zeros((1, 2, 3), np.int64)), freq),
            lambda: turn(x, put(sp, np.zeros(3, F32)), freq),
            lambda: turn(x, sp.Tensor.from_numpy(np.arange(3)), freq),
            lambda: turn(x, positions, put(sp, np.zeros(4, F32))),
            lambda: turn(x, positions, put(sp, np.zeros(5))),
            lambda: turn(x, positions, sp.rotary_frequencies(8)),
            lambda: turn(x, positions, put(sp, oracle.frequencies(8), grad=True)),
            lambda: turn(x, positions, freq, magnitude=nan),
            lambda: norm(x, double, weight, weight, positions, freq),
            lambda: norm(x, put(sp, np.zeros((2, 4, 4, 8), F32)), weight, weight, positions, freq),
            lambda: norm(x, x, put(sp, np.ones(7, F32)), weight, positions, freq),
            lambda: norm(x, x, weight, put(sp, np.ones(8)), positions, freq),
            lambda: norm(x, x, weight, weight, positions, freq, epsilon=0.0),
            lambda: norm(wide, wide, put(sp, np.ones(258, F32)), put(sp, np.ones(258, F32)),
                         put(sp, np.arange(1)), freq),
            lambda: attend(x, three, three),
            lambda: attend(x, x, three),
            lambda: attend(x, double, double),
            lambda: attend(x, wide, wide),
            lambda: attend(wide, wide, wide),
            lambda: attend(x, x, x, scale=nan),
            lambda: attend(x, x, x, lengths=put(sp, np.zeros(3, np.int32))),
            lambda: attend(x, x, x, lengths=put(sp, np.zeros(2, F32))),
            lambda: attend(x, x, x, lengths=sp.Tensor.from_numpy(np.zeros(2, np.int32)))):
        with pytest.raises(ValueError):
            call()


def test_backward_keeps_positions_and_lengths_as_they_were(sp):
    """A program that counts its positions and lengths on between forward and backward."""
    rng = np.random.default_rng(17)
    x = rng.standard_normal((2, 2, 9, 32))

    def gradient(changes):
        leaf = put(sp, x, grad=True)
        weight = put(sp, np.ones(32), grad=True)
        positions, lengths = put(sp, np.arange(9)), put(sp, np.array([9, 6]))
        freq = put(sp, oracle.frequencies(32))
        turned = sp.rotary_embedding(leaf, positions, freq)
        query, key = sp.query_key_norm_rotary(turned, turned, weight, weight, positions, freq)
        out = sp.window_attention(query, key, turned, 4, 1, lengths=lengths)
        if changes:
            sp.copy_values(positions, put(sp, np.arange(9) + 100))
            sp.copy_values(lengths, put(sp, np.array([1, 1])))
        sp.sum(sp.multiply(out, out)).backward()
        return get(sp, leaf.grad()), get(sp, weight.grad())

    for a, b in zip(gradient(False), gradient(True)):
        assert np.array_equal(a, b)


def test_results_after_the_inputs_are_gone(sp):
    """A graph keeps what its backward reads, although the program drops it."""
    rng = np.random.default_rng(16)
    x = rng.standard_normal((1, 2, 50, 64))
    leaf = put(sp, x, grad=True)

    def loss():
        made = sp.rotary_embedding(leaf, put(sp, np.arange(50)), put(sp, oracle.frequencies(64)))
        out = sp.window_attention(made, made, made, 9, 2, lengths=put(sp, np.array([41])))
        return sp.sum(sp.multiply(out, out))

    first = loss()
    for _ in range(4):
        put(sp, rng.standard_normal((1, 2, 50, 64)))  # takes over what was freed
    first.backward()
    kept = get(sp, leaf.grad())
    leaf.zero_grad()
    loss().backward()
    assert np.array_equal(kept, get(sp, leaf.grad()))
