"""What the attention operators refuse on the host, and rotary frequencies: no GPU."""
import ctypes
import math

import numpy as np
import pytest

from spar_amd import hip, spar

A, B = 1 << 20, 1 << 21  # addresses that are never read: every call is refused or empty


def heads(address=A):
    return hip.heads(address, (64, 64, 64))


def rotary(**changes):
    values = dict(positions=A, position_stride=0, position_dtype=hip.INT32, frequencies=A,
                  rotary_extent=64, magnitude=1.0, layout=0)
    return hip.rotary(**(values | changes))


def turn(output=None, source=None, batch=1, count=1, tokens=1, extent=64, rotation=None, inverse=0,
         dtype=0):
    return hip.status_of("spar_hip_launch_rotary", output or heads(), source or heads(), batch,
                         count, tokens, extent, rotation or rotary(), inverse, dtype, 0).code


@pytest.mark.parametrize("changes", [
    dict(dtype=2), dict(inverse=2), dict(extent=62), dict(output=heads(None)),
    dict(source=heads(None)), dict(rotation=rotary(rotary_extent=63)),
    dict(rotation=rotary(layout=2)), dict(rotation=rotary(position_dtype=0)),
    dict(rotation=rotary(magnitude=math.inf)), dict(rotation=rotary(magnitude=math.nan)),
    dict(rotation=rotary(positions=None)), dict(rotation=rotary(frequencies=None)),
    dict(count=1 << 30), dict(batch=1 << 40, tokens=1 << 39),
], ids=str)
def test_rotary_refuses(changes):
    assert turn(**changes) == 1


@pytest.mark.parametrize("changes", [dict(batch=0), dict(count=0), dict(tokens=0)], ids=str)
def test_rotary_of_nothing_succeeds(changes):
    assert turn(output=heads(None), source=heads(None), **changes) == 0


def norm_forward(parts=None, count=1, batch=1, tokens=1, extent=64, rotation=None, epsilon=1e-5,
                 dtype=0, **part):
    values = dict(output=A, source=A, weight=A, heads=2) | part
    made = hip.head_norms(*[(values["output"], (1, 1, 1), None, values["source"], (1, 1, 1),
                             values["weight"], values["heads"])] * 2)
    return hip.status_of("spar_hip_launch_head_norm_rotary_forward", made, count, batch, tokens,
                         extent, rotation or rotary(), epsilon, dtype, 0).code


@pytest.mark.parametrize("changes", [
    dict(count=0), dict(count=3), dict(extent=0), dict(extent=257), dict(dtype=3),
    dict(epsilon=0.0), dict(epsilon=math.nan), dict(epsilon=math.inf), dict(output=None),
    dict(source=None), dict(weight=None), dict(rotation=rotary(rotary_extent=66)),
], ids=str)
def test_head_norm_refuses(changes):
    assert norm_forward(**changes) == 1


def test_head_norm_refuses_too_many_heads_in_all():
    assert norm_forward(heads=(1 << 24) - 1, count=2) == 1


def test_head_norm_of_nothing_succeeds():
    assert norm_forward(tokens=0, output=None) == 0
    assert norm_forward(heads=0, output=None) == 0


def test_head_norm_backward_refuses_a_small_workspace():
    need = hip.head_norm_rotary_workspace(2, 100, 3, 64, 0)
    assert need == 75 * 2 * 64 * 4  # a partial row for each 8 heads

    def status(workspace, size, weight_gradient=A):
        part = hip.head_norm_gradients((A, (1, 1, 1), weight_gradient, A, (1, 1, 1), A, (1, 1, 1),
                                        A, A, 3))
        return hip.status_of("spar_hip_launch_head_norm_rotary_backward", part, 1, 2, 100, 64,
                             rotary(), workspace, size, 0, 0).code

    assert status(None, need) == 1
    assert status(B, need - 1) == 1
    assert status(B + 4, need) == 1
    assert status(B, need, None) == 1


def attention(**changes):
    values = dict(batch=2, query_heads=4, key_heads=2, queries=8, keys=8, extent=64, window=4,
                  sinks=1, scale=0.125, lengths=None, length_dtype=hip.INT32, dtype=0)
    return hip.attention(**(values | changes))


def forward(shape, output=A, query=A, key=A, value=A, workspace=None, size=0):
    return hip.status_of("spar_hip_launch_attention_forward", heads(output), None, heads(query),
                         heads(key), heads(value), shape, workspace, size, 0).code


BAD_SHAPES = [dict(key_heads=0), dict(query_heads=0), dict(query_heads=3), dict(extent=0),
              dict(extent=257), dict(dtype=2), dict(scale=math.inf), dict(scale=math.nan),
              dict(keys=1 << 30), dict(queries=1 << 28), dict(batch=1 << 31),
              dict(lengths=A, length_dtype=0)]


@pytest.mark.parametrize("changes", BAD_SHAPES, ids=str)
def test_attention_refuses_shapes(changes):
    need = ctypes.c_uint64(0)
    for backward in (0, 1):
        assert hip.status_of("spar_hip_attention_workspace", ctypes.byref(need),
                             attention(**changes), backward).code == 1
    assert forward(attention(**changes)) == 1


@pytest.mark.parametrize("which", ["output", "query", "key", "value"])
def test_attention_refuses_missing_tensors(which):
    assert forward(attention(), **{which: None}) == 1


def test_attention_refuses_small_workspaces():
    shape = attention(queries=1, keys=65536, window=0)
    need = hip.attention_workspace(shape, 0)
    assert need > 0
    assert forward(shape, workspace=None, size=need) == 1
    assert forward(shape, workspace=B, size=need - 1) == 1
    assert forward(shape, workspace=B + 8, size=need) == 1
    shape = attention()
    need = hip.attention_workspace(shape, 1)
    for workspace, size, logsumexp in ((None, need, A), (B, need - 1, A), (B + 8, need, A),
                                       (B, need, None)):
        assert hip.status_of("spar_hip_launch_attention_backward", *[heads()] * 5, logsumexp,
                             *[heads()] * 3, shape, workspace, size, 0).code == 1
    assert hip.status_of("spar_hip_attention_workspace", None, shape, 0).code == 1
    assert hip.status_of("spar_hip_attention_workspace", ctypes.byref(ctypes.c_uint64()), shape,
                         2).code == 1


def test_parts_of_many_sinks_stay_bounded():
    """A tile of 64 sinks has a part [2, 64, extent] for each split of its later rows;
    2048 such parts at most once the tiles are many."""
    shape = attention(batch=1, query_heads=8, key_heads=8, queries=131071, keys=131071,
                      extent=128, window=1024, sinks=4096)
    parts = hip.attention_workspace(shape, 1) - 8 * 131071 * 4 // 16 * 16
    assert 0 < parts <= 2048 * 2 * 64 * 128 * 4 + 16


def test_attention_of_nothing_succeeds():
    assert forward(attention(batch=0), output=None, query=None) == 0
    assert forward(attention(queries=0), output=None, query=None) == 0


# -------------------------------------------------------------- frequencies

def test_rotary_frequencies():
    """Against the formulas in numpy's doubles: a power and two products, each of at
    most 2 steps."""
    j = np.arange(16)
    plain = 500.0 ** (-2.0 * j / 32)
    near = dict(rtol=8 * np.finfo(float).eps, atol=0)
    np.testing.assert_allclose(spar.rotary_frequencies(32, 500.0).numpy(), plain, **near)
    kind, scaling = spar.RotaryScaling.Kind, spar.RotaryScaling
    np.testing.assert_allclose(
        spar.rotary_frequencies(32, 500.0, scaling(kind.Linear, 4.0)).numpy(), plain / 4, **near)
    stretched = spar.rotary_frequencies(32, 500.0, scaling(kind.Base, 4.0)).numpy()
    assert stretched[0] == 1.0
    np.testing.assert_allclose(stretched[-1], plain[-1] / 4, rtol=1e-14)
    parts = spar.rotary_frequencies(32, 500.0, scaling(kind.Parts, 4.0, 1000.0, 1.0, 8.0)).numpy()
    keep = np.clip((1000 * plain / (2 * np.pi) - 1) / 7, 0, 1)
    np.testing.assert_allclose(parts, plain * keep + plain / 4 * (1 - keep), rtol=1e-14)
    assert 0 < keep[(keep > 0) & (keep < 1)].size < 16 and keep[0] == 1
    assert spar.rotary_magnitude(4.0) == pytest.approx(0.1 * math.log(4) + 1, rel=1e-15)


@pytest.mark.parametrize("arguments", [
    (0,), (7,), (8, 0.0), (8, math.inf), (8, 10.0, ("Linear", 0.0)), (2, 10.0, ("Base", 2.0)),
    (8, 10.0, ("Parts", 2.0)), (8, 10.0, ("Parts", 2.0, 100.0, 8.0, 8.0)),
    (8, 10.0, ("Parts", 2.0, 100.0, 1.0, math.inf)),
], ids=str)
def test_rotary_frequencies_refuses(arguments):
    if len(arguments) == 3:
        name, *rest = arguments[2]
        arguments = (*arguments[:2],
                     spar.RotaryScaling(getattr(spar.RotaryScaling.Kind, name), *rest))
    with pytest.raises(ValueError):
        spar.rotary_frequencies(*arguments)
    with pytest.raises(ValueError):
        spar.rotary_magnitude(-1.0)


def test_operators_need_hip_tensors_of_the_right_shapes():
    x = spar.Tensor.from_numpy(np.zeros((1, 2, 3, 4), np.float32))
    positions = spar.Tensor.from_numpy(np.arange(3))
    freq = spar.rotary_frequencies(4)
    weight = spar.Tensor.from_numpy(np.ones(4, np.float32))
    with pytest.raises(RuntimeError):
        spar.rotary_embedding(x, positions, freq)
    with pytest.raises(RuntimeError):
        spar.query_key_norm_rotary(x, x, weight, weight, positions, freq)
    with pytest.raises(RuntimeError):
        spar.window_attention(x, x, x)
    flat = spar.Tensor.from_numpy(np.zeros((3, 4), np.float32))
    whole = spar.Tensor.from_numpy(np.zeros((1, 2, 3, 4), np.int32))
    for wrong in (flat, whole):
        with pytest.raises(ValueError):
            spar.rotary_embedding(wrong, positions, freq)
        with pytest.raises(ValueError):
            spar.window_attention(wrong, wrong, wrong)
