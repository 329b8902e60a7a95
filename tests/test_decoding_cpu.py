"""What the decoding operators refuse on the host, their workspaces, and calls of nothing:
no GPU."""
import ctypes
import math

import numpy as np
import pytest

from spar_amd import hip, spar

A = 1 << 20  # an address that is never read
NO_DEVICE = 999  # calls that pass the checks end here


def heads(address=A):
    return hip.heads(address, (64, 64, 64))


def pages(key=A, value=A, count=8, page_tokens=16, table=A, table_stride=4, table_pages=4):
    return hip.pages(key, (64, 64, 64), value, (64, 64, 64), count, page_tokens, table,
                     table_stride, table_pages)


def rotary(**changes):
    values = dict(positions=A, position_stride=0, position_dtype=hip.INT32, frequencies=A,
                  rotary_extent=64, magnitude=1.0, layout=0)
    return hip.rotary(**(values | changes))


# ------------------------------------------------------------------- append

def append(cache=None, output=heads(), query=heads(), query_heads=4, key=heads(), value=heads(),
           batch=2, key_heads=2, tokens=3, extent=64, places=A, place_dtype=hip.INT32,
           rotation=rotary(), dtype=0, device=NO_DEVICE):
    return hip.status_of("spar_hip_launch_cache_append", cache or pages(), output, query,
                         query_heads, key, value, batch, key_heads, tokens, extent, places, 3,
                         place_dtype, rotation, dtype, device).code


@pytest.mark.parametrize("changes", [
    dict(dtype=2), dict(place_dtype=0), dict(cache=pages(page_tokens=0)),
    dict(cache=pages(table_pages=1 << 27)), dict(cache=pages(page_tokens=1 << 30)),
    dict(cache=pages(page_tokens=1 << 40, table_pages=1 << 30)),
    dict(cache=pages(table=None, table_pages=2)), dict(cache=pages(key=None)),
    dict(cache=pages(value=None)), dict(output=None), dict(query=None), dict(output=heads(None)),
    dict(query=heads(None)), dict(key=None), dict(value=None), dict(key=heads(None)),
    dict(value=heads(None)), dict(places=None), dict(rotation=rotary(rotary_extent=63)),
    dict(rotation=rotary(rotary_extent=66)), dict(rotation=rotary(layout=2)),
    dict(rotation=rotary(positions=None)), dict(rotation=rotary(frequencies=None)),
    dict(rotation=rotary(magnitude=math.nan)), dict(key_heads=1 << 24),
    dict(query_heads=1 << 30), dict(batch=1 << 31), dict(batch=1 << 30, tokens=1 << 39),
    dict(extent=1 << 23, key_heads=1 << 20, rotation=None),
], ids=str)
def test_append_refuses(changes):
    assert append(**changes) == 1


@pytest.mark.parametrize("changes", [
    dict(batch=0), dict(tokens=0), dict(extent=0, rotation=None),
    dict(key_heads=0, query=None, output=None),
], ids=str)
def test_append_of_nothing_succeeds(changes):
    assert append(**changes) == 0


@pytest.mark.parametrize("changes", [
    {}, dict(query=None, output=None), dict(rotation=None), dict(place_dtype=hip.INT64),
    dict(cache=pages(key=None, value=None, count=0)),
    dict(cache=pages(key=None, value=None, table_pages=0)),
    dict(cache=pages(table=None, table_pages=1)),
    dict(key_heads=0, key=None, value=None, places=None),
], ids=str)
def test_append_takes(changes):
    assert append(**changes) not in (0, 1)


# ---------------------------------------------------------------- attention

def shape(batch=4, prefixes=2, query_heads=4, key_heads=2, queries=1, extent=64, scale=1.0,
          lengths=A, prefix_lengths=A, length_dtype=hip.INT32, dtype=0):
    return hip.cache_attention(batch, prefixes, query_heads, key_heads, queries, extent, scale,
                               lengths, prefix_lengths, length_dtype, dtype)


NONE = object()


def attend(call=None, cache=None, prefix=None, output=heads(), query=heads(), workspace=A,
           short=0):
    cache = cache or pages()
    prefix = None if prefix is NONE else prefix or pages()
    call = call or shape()
    need = ctypes.c_uint64(0)
    status = hip.status_of("spar_hip_cache_attention_workspace", ctypes.byref(need), cache, prefix,
                           call).code
    done = hip.status_of("spar_hip_launch_cache_attention", output, query, cache, prefix, call,
                         workspace, max(0, need.value - short), NO_DEVICE).code
    assert status == 0 or done == 1
    return done


@pytest.mark.parametrize("changes", [
    dict(dtype=2), dict(key_heads=0), dict(query_heads=0), dict(query_heads=5), dict(extent=0),
    dict(extent=257), dict(scale=math.inf), dict(scale=math.nan), dict(prefixes=0),
    dict(prefixes=3), dict(length_dtype=0), dict(batch=1 << 31), dict(batch=1 << 30),
    dict(queries=1 << 31), dict(queries=1 << 28), dict(batch=1 << 23, prefixes=1, queries=64),
    dict(batch=1 << 29, prefixes=1),
], ids=str)
def test_attention_refuses(changes):
    assert attend(shape(**changes)) == 1


@pytest.mark.parametrize("changes", [
    dict(output=None), dict(query=None), dict(output=heads(None)), dict(query=heads(None)),
    dict(workspace=None), dict(workspace=A + 4), dict(short=1), dict(cache=pages(key=None)),
    dict(cache=pages(page_tokens=0)), dict(prefix=pages(value=None)),
    dict(prefix=pages(page_tokens=1 << 29, table_pages=2)),
    dict(prefix=pages(table=None, table_pages=3)),
], ids=str)
def test_attention_refuses_buffers(changes):
    assert attend(**changes) == 1


@pytest.mark.parametrize("changes", [dict(batch=0), dict(queries=0)], ids=str)
def test_attention_of_nothing_succeeds(changes):
    assert attend(shape(**changes), output=None, query=None) == 0


@pytest.mark.parametrize("call,more", [
    (shape(), {}), (shape(length_dtype=0, lengths=None, prefix_lengths=None), {}),
    (shape(prefixes=0), dict(prefix=NONE)), (shape(batch=3, prefixes=2), dict(prefix=NONE)),
    (shape(), dict(cache=pages(key=None, value=None, count=0))),
    (shape(), dict(prefix=pages(table=None, table_pages=1, page_tokens=1000))),
], ids=str)
def test_attention_takes(call, more):
    assert attend(call, **more) not in (0, 1)


def test_attention_workspace():
    """One part needs none; otherwise each row of each part its values, base and sum."""
    one = pages(page_tokens=64, table_pages=1)
    assert hip.cache_attention_workspace(one, None, shape()) == 0
    need = hip.cache_attention_workspace(one, one, shape(extent=62))
    assert need == 2 * 16 * (64 + 2) * 4
    assert hip.cache_attention_workspace(one, one, shape(extent=62, dtype=1)) == 2 * 16 * 64 * 8
    assert hip.status_of("spar_hip_cache_attention_workspace", None, one, None, shape()).code == 1


# -------------------------------------------------------------------- beams

def beams(groups=2, count=3, vocabulary=100, picks=4, row_stride=100, ended=None, end_token=-1,
          dtype=0):
    return hip.beams(groups, count, vocabulary, picks, row_stride, ended, end_token, dtype)


def select(call=None, short=0, **changes):
    call = call or beams()
    need = ctypes.c_uint64(0)
    hip.status_of("spar_hip_beam_select_workspace", ctypes.byref(need), call)
    values = dict(scores=A, parents=A, tokens=A, flags=None, logits=A, before=A,
                  workspace=A) | changes
    return hip.status_of("spar_hip_launch_beam_select", values["scores"], values["parents"],
                         values["tokens"], values["flags"], values["logits"], values["before"],
                         call, values["workspace"], max(0, need.value - short), NO_DEVICE).code


@pytest.mark.parametrize("changes", [
    dict(dtype=2), dict(count=0), dict(count=65), dict(picks=0), dict(picks=65),
    dict(vocabulary=0), dict(vocabulary=1 << 31, row_stride=1 << 31), dict(row_stride=99),
    dict(count=1, vocabulary=3, picks=4), dict(groups=1 << 24), dict(groups=1 << 60),
    dict(end_token=100), dict(ended=A, end_token=-1), dict(ended=A, end_token=100),
], ids=str)
def test_select_refuses(changes):
    assert select(beams(**changes)) == 1


@pytest.mark.parametrize("changes", [
    dict(scores=None), dict(parents=None), dict(tokens=None), dict(logits=None),
    dict(before=None), dict(workspace=None), dict(workspace=A + 8), dict(short=1),
], ids=str)
def test_select_refuses_buffers(changes):
    assert select(**changes) == 1


def test_select_takes():
    assert select(beams(groups=0), scores=None) == 0
    assert select() not in (0, 1)
    assert select(beams(ended=A, end_token=99, picks=64, count=64), flags=A) not in (0, 1)


def move(*states, parents=A, rows=4, source_rows=4, count=None):
    made = hip.reorders(*states)
    return hip.status_of("spar_hip_launch_reorder", made, len(states) if count is None else count,
                         parents, rows, source_rows, NO_DEVICE).code


@pytest.mark.parametrize("state,changes", [
    ((A, 8, A, 8, 8, 2), {}), ((A, 8, A, 8, 8, 16), {}), ((A, 7, A, 8, 8, 4), {}),
    ((None, 8, A, 8, 8, 4), {}), ((A, 8, None, 8, 8, 4), {}), ((A, 8, A, 8, 8, 4),
                                                               dict(parents=None)),
    ((A, 8, A, 8, 8, 4), dict(rows=1 << 31)), ((A, 8, A, 8, 8, 4), dict(rows=1 << 24)),
    ((A, 1 << 49, A, 8, 8, 4), {}), ((A, 8, A, 1 << 49, 8, 4), {}),
    ((A, 8, A, 8, 8, 4), dict(count=(1 << 16) + 1)),
], ids=str)
def test_reorder_refuses(state, changes):
    assert move(state, **changes) == 1


@pytest.mark.parametrize("elements,rows", [(1 << 48, 1 << 27), (1 << 47, 1 << 28), (1 << 41, 4)])
def test_reorder_refuses_more_than_its_products_hold(elements, rows):
    # 2^48 elements of 8 bytes are 2^37 workgroups of 2^14 bytes a row: 2^64 in all
    assert move((A, elements, A, elements, elements, 8), rows=rows) == 1


def test_reorder_takes():
    assert move() == 0
    assert move((A, 8, A, 8, 8, 4), rows=0, parents=None) == 0
    assert move((A, 8, A, 8, 8, 4)) not in (0, 1)
    assert move((A, 8, None, 8, 8, 8), source_rows=0) not in (0, 1)


# --------------------------------------------------------------- tensor API

def cpu(shape, kind=np.float32):
    return spar.Tensor.from_numpy(np.zeros(shape, kind))


def test_host_tensors_are_refused():
    x = cpu((1, 2, 3, 8))
    cache = spar.PagedCache(x, x)
    with pytest.raises(RuntimeError, match="HIP tensor"):
        spar.cache_append(cache, x, x, cpu((1, 3), np.int32))
    with pytest.raises(RuntimeError, match="HIP tensor"):
        spar.cache_attention(x, cache)
    with pytest.raises(RuntimeError, match="HIP tensor"):
        spar.beam_select(cpu((1, 2, 3)), cpu((1, 2)), 2)
    with pytest.raises(RuntimeError, match="HIP tensor"):
        spar.reorder([x], cpu((3,), np.int64))


def test_wrong_ranks_and_types_are_refused():
    x = cpu((1, 2, 3, 8))
    with pytest.raises(ValueError, match="batch, heads, tokens, extent"):
        spar.cache_attention(cpu((2, 3, 8)), spar.PagedCache(x, x))
    with pytest.raises(ValueError, match="floating-point"):
        spar.cache_attention(cpu((1, 2, 3, 8), np.int32), spar.PagedCache(x, x))
    with pytest.raises(ValueError, match="groups, beams, vocabulary"):
        spar.beam_select(cpu((2, 3)), cpu((2, 3)), 1)
    with pytest.raises(ValueError, match="Int64"):
        spar.reorder([x], cpu((3,), np.int32))
