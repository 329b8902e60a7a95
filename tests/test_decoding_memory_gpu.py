"""The decoding operators and what memory holds: workspaces and outputs full of NaN before
the call, and caches whose elements lie more than 2^32 from their start."""
import numpy as np
import pytest

from tests import decoding_oracle as oracle
from tests import test_beams_gpu as beams
from tests import test_cache_attention_gpu as attention
from tests.test_cache_attention_gpu import assert_within, random

pytestmark = pytest.mark.gpu

F32, F64 = np.float32, np.float64


@pytest.fixture(autouse=True)
def _release_buffers():
    yield
    attention._alive.clear()
    beams._alive.clear()


@pytest.fixture
def undefined(monkeypatch):
    """Workspaces and outputs come as NaN (and as numbers no parent or token has)."""
    for module in (attention, beams):
        monkeypatch.setattr(module, "space", lambda hip, nbytes, module=module: module.device(
            hip, np.full(max(int(nbytes), 16), 255, np.uint8)))


@pytest.mark.parametrize("dtype", [F32, F64])
@pytest.mark.parametrize("case", [  # (batch, heads, key heads, queries, room, extent), lengths,
    # page, prefix, its lengths, its page
    ((6, 8, 2, 1, 700, 64), [700, 0, 1, 64, 65, 300], 16, (2, 1000), [1000, 0], 0),
    ((6, 8, 1, 1, 700, 72), [700, 0, 1, 64, 65, 300], 5, (3, 500), [0, 500, 1], 7),
    ((4, 4, 1, 40, 300, 128), [300, 10, 0, 41], 32, (1, 600), [600], 64),
], ids=str)
def test_attention_workspaces_may_hold_anything(hip, undefined, case, dtype):
    shape, lengths, page, prefix, prefix_lengths, prefix_page = case
    attention.check(hip, shape, dtype, lengths, page, prefix, prefix_lengths, prefix_page)


@pytest.mark.parametrize("dtype", [F32, F64])
@pytest.mark.parametrize("picks", [3, 64])
def test_selection_workspaces_may_hold_anything(hip, undefined, picks, dtype):
    logits, scores = beams.inputs(3, 4, 9001, dtype, 32)
    logits[0, 1] = -np.inf  # a row without a candidate
    ended = np.zeros((3, 4), np.int32)
    ended[1] = 1            # a group whose rows are not read
    ended[2, 3] = 1
    beams.check(hip, logits, scores, picks, ended, 17)


@pytest.mark.parametrize("page", [128, 5])
@pytest.mark.parametrize("heads,queries", [(2, 1), (8, 1), (8, 770)])
def test_attention_far_into_a_large_cache(hip, page, heads, queries):
    """Few rows, 16 rows and tiles over pages more than 2^32 elements from the cache's start,
    as a prefix and as the sequences' own."""
    b, hk, d, n = 2, 1, 128, 800
    entries = -(-n // page)
    pages = 5 * 2 ** 30 // (page * d)
    count = pages * page * d
    assert count > 2 ** 32
    key, value = (attention.space(hip, 4 * count) for _ in range(2))
    # rows 0 and 1 are the sequences', row 2 the prefix's, all in the last pages
    numbers = np.random.default_rng(3).permutation(np.arange(pages - 3 * entries, pages))
    numbers = numbers.reshape(3, entries).astype(np.int32)
    assert int(numbers.min()) * page * d > 2 ** 32
    table = attention.device(hip, numbers)
    strides = (page * d, page * d, d)
    cache = hip.pages(key.ptr, strides, value.ptr, strides, pages, page, table.ptr, entries,
                      entries)
    prefix = hip.pages(key.ptr, strides, value.ptr, strides, pages, page,
                       table.address(4 * 2 * entries), entries, entries)
    keys, values = random((3, hk, n, d), F32, 1), random((3, hk, n, d), F32, 2)
    places = attention.device(hip, np.broadcast_to(np.arange(n), (3, n)).astype(np.int32))
    hip.call("spar_hip_launch_cache_append", cache, None, None, 0,
             attention.Heads(hip, keys).heads, attention.Heads(hip, values).heads, 3, hk, n, d,
             places.ptr, n, hip.INT32, None, 0, 0)
    query, lengths = random((b, heads, queries, d), F32, 3), [n, n - 13]
    output = attention.Heads(hip, np.full_like(query, 5.0))
    shape = hip.cache_attention(
        b, 1, heads, hk, queries, d, 1 / np.sqrt(d),
        attention.device(hip, np.array(lengths, np.int32)).ptr,
        attention.device(hip, np.array([n], np.int32)).ptr, hip.INT32, 0)
    need = hip.cache_attention_workspace(cache, prefix, shape)
    hip.call("spar_hip_launch_cache_attention", output.heads,
             attention.Heads(hip, query).heads, cache, prefix, shape,
             attention.space(hip, need).ptr, need, 0)
    want, bound = oracle.attention(query, oracle.Pool(keys[:2], values[:2], lengths, 0), lengths,
                                   oracle.Pool(keys[2:], values[2:], [n], 0), [n], None, F32)
    assert_within(output.numpy(), want, bound)
    del key, value
    attention._alive.clear()
    hip.call("spar_hip_empty_cache", 0)


@pytest.mark.parametrize("shared", [False, True])
def test_attention_of_more_rows_than_a_launch_has_workgroups(hip, shared):
    """2^24 rows and more, of which the last of every sequence see something: without a prefix
    and behind one, whose parts a second launch joins."""
    b, h, hk, t, n, d = 64, 8, 2, 32800, 20, 4
    rows = b * h * t
    assert rows > 2 ** 24
    lengths = [n - i % 4 for i in range(b)]
    cache = attention.Cache(hip, oracle.Pool(random((b, hk, n, d), F32, 1),
                                             random((b, hk, n, d), F32, 2), lengths, 4))
    pool = oracle.Pool(random((2, hk, 30, d), F32, 3), random((2, hk, 30, d), F32, 4), [30, 7], 0)
    prefix = attention.Cache(hip, pool).pages if shared else None
    seen = random((b, h, n, d), F32, 5)  # the queries that see something, and others
    query = attention.space(hip, 4 * rows * d)
    hip.call("spar_hip_launch_fill", query.ptr, rows * d, 0, 1.0, 0)
    for i in range(b):
        for j in range(h):
            at = query.ptr + 4 * d * ((i * h + j) * t + t - n)
            hip.call("spar_hip_copy_host_to_device", at,
                     np.ascontiguousarray(seen[i, j]).ctypes.data, 4 * n * d, 0)
    output = attention.space(hip, 4 * rows * d)
    hip.call("spar_hip_launch_fill", output.ptr, rows * d, 0, 3.0, 0)
    strides = (h * t * d, t * d, d)
    shape = hip.cache_attention(
        b, 2, h, hk, t, d, 0.5, attention.device(hip, np.array(lengths, np.int32)).ptr,
        attention.device(hip, np.array([30, 7], np.int32)).ptr if shared else None, hip.INT32, 0)
    need = hip.cache_attention_workspace(cache.pages, prefix, shape)
    assert need == (2 * rows * (d + 2) * 4 if shared else 0)
    workspace = attention.space(hip, need)
    hip.call("spar_hip_launch_cache_attention", hip.heads(output.ptr, strides),
             hip.heads(query.ptr, strides), cache.pages, prefix, shape, workspace.ptr, need, 0)
    got = output.to_numpy(F32, (b, h, t, d))
    assert not got[:, :, :t - n].any()
    want, bound = oracle.attention(seen, cache.pool, lengths, pool if shared else None,
                                   [30, 7] if shared else None, 0.5, F32)
    assert_within(got[:, :, t - n:], want, bound)
    del query, output, workspace
    attention._alive.clear()
    hip.call("spar_hip_empty_cache", 0)
