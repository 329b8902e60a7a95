"""The paged cache and attention over it behind a shared prefix, through the C ABI, against
their definitions in 64 bits."""
import ctypes

import numpy as np
import pytest

from tests import attention_oracle, decoding_oracle as oracle
from tests.attention_oracle import assert_within, half_step

pytestmark = pytest.mark.gpu

F32, F64 = np.float32, np.float64
_alive = []


@pytest.fixture(autouse=True)
def _release_buffers():
    yield
    _alive.clear()


def device(hip, array):
    buffer = hip.DeviceBuffer.from_numpy(np.ascontiguousarray(array))
    _alive.append(buffer)
    return buffer


def space(hip, nbytes):
    buffer = hip.DeviceBuffer(max(int(nbytes), 16))
    _alive.append(buffer)
    return buffer


class Heads:
    """[batch, heads, tokens, extent] values as [batch, tokens, heads, extent + gap]."""

    def __init__(self, hip, values, gap=0, offset=0, fill=0.0):
        b, h, t, d = values.shape
        self.shape, self.gap, self.offset = values.shape, gap, offset
        whole = np.full(offset + b * t * h * (d + gap), fill, values.dtype)
        rows = whole[offset:].reshape(b, t, h, d + gap)
        rows[..., :d] = values.transpose(0, 2, 1, 3)
        self.count, self.dtype, self.buffer = whole.size, values.dtype, device(hip, whole)
        self.strides = (t * h * (d + gap), d + gap, h * (d + gap))
        self.heads = hip.heads(self.buffer.address(offset * values.dtype.itemsize), self.strides)

    def numpy(self):
        b, h, t, d = self.shape
        whole = self.buffer.to_numpy(self.dtype, (self.count,))
        rows = whole[self.offset:].reshape(b, t, h, d + self.gap)
        self.gaps = rows[..., d:]
        return rows[..., :d].transpose(0, 2, 1, 3)


class Cache:
    """A Pool on the device, [page, head, token, extent + gap] or, `interleaved`, keys and
    values side by side as [page, token, 2, head, extent + gap]."""

    def __init__(self, hip, pool, gap=0, offset=0, interleaved=False, entries=None):
        self.pool, self.gap, self.offset, self.interleaved = pool, gap, offset, interleaved
        n, h, p, d = pool.key.shape
        both = np.stack([pool.key, pool.value])  # [2, page, head, token, extent]
        order = (1, 3, 0, 2, 4) if interleaved else (0, 1, 2, 3, 4)
        outer = both.transpose(order)
        whole = np.full(offset + outer[..., 0].size * (d + gap), 7.0, both.dtype)
        whole[offset:].reshape(*outer.shape[:-1], d + gap)[..., :d] = outer
        self.outer, self.order, self.dtype = outer.shape, order, both.dtype
        self.buffer, self.count = device(hip, whole), whole.size
        size = both.dtype.itemsize
        w = d + gap
        strides = (p * 2 * h * w, w, 2 * h * w) if interleaved else (h * p * w, p * w, w)
        step = h * w if interleaved else n * h * p * w
        table = pool.table
        self.table = None if table is None else device(hip, table)
        self.pages = hip.pages(self.buffer.address(offset * size), strides,
                               self.buffer.address((offset + step) * size), strides, n,
                               pool.page_tokens, None if table is None else self.table.ptr,
                               0 if table is None else table.shape[1],
                               1 if table is None else
                               (table.shape[1] if entries is None else entries))

    def numpy(self):
        """(keys, values) [page, head, token, extent]."""
        d = self.outer[-1]
        whole = self.buffer.to_numpy(self.dtype, (self.count,))
        rows = whole[self.offset:].reshape(*self.outer[:-1], d + self.gap)
        self.gaps = rows[..., d:]
        return rows[..., :d].transpose(np.argsort(self.order))


def attend(hip, query, cache, lengths=None, prefix=None, prefix_lengths=None, scale=None,
           length_type=np.int32, gap=0, offset=0, **layout):
    b, h, t, d = query.shape
    dtype = hip.dtype_tag(query.dtype)
    output = Heads(hip, np.full_like(query, 5.0), gap, offset)
    q = Heads(hip, query, gap, offset)
    own = Cache(hip, cache, **layout)
    shared = None if prefix is None else Cache(hip, prefix, **layout)

    def counted(values):
        return None if values is None else device(hip, np.asarray(values, length_type)).ptr

    shape = hip.cache_attention(b, 1 if prefix is None else prefix.rows, h, cache.heads, t, d,
                                1 / np.sqrt(d) if scale is None else scale, counted(lengths),
                                counted(prefix_lengths), hip.dtype_tag(length_type), dtype)
    pages = None if shared is None else shared.pages
    need = hip.cache_attention_workspace(own.pages, pages, shape)
    hip.call("spar_hip_launch_cache_attention", output.heads, q.heads, own.pages, pages, shape,
             space(hip, need).ptr if need else None, need, 0)
    got = output.numpy()
    assert not output.gaps.any()
    return got


def random(shape, dtype, seed):
    return np.random.default_rng(seed).standard_normal(shape).astype(dtype)


def check(hip, shape, dtype, lengths, page, prefix=None, prefix_lengths=None, prefix_page=0,
          scale=None, **more):
    """shape: batch, heads, key heads, queries, own room, extent; prefix: rows, room."""
    b, h, hk, t, n, d = shape
    query = random((b, h, t, d), dtype, 1)
    cache = oracle.Pool(random((b, hk, n, d), dtype, 2), random((b, hk, n, d), dtype, 3), lengths,
                        page)
    shared = None
    if prefix is not None:
        rows, room = prefix
        full = [room] * rows if prefix_lengths is None else prefix_lengths
        if room == 0 or (prefix_page and room % prefix_page):  # pages have room for more
            prefix_lengths = full
        shared = oracle.Pool(random((rows, hk, room, d), dtype, 4),
                             random((rows, hk, room, d), dtype, 5), full, prefix_page, seed=6)
    want, bound = oracle.attention(query, cache, lengths, shared, prefix_lengths, scale, dtype)
    got = attend(hip, query, cache, lengths, shared, prefix_lengths, scale, **more)
    assert_within(got, want, bound)
    return got


CASES = [  # (batch, heads, key heads, queries, room, extent), lengths, page, prefix, its lengths, page
    ((1, 1, 1, 1, 1, 1), [1], 1, None, None, 0),
    ((2, 2, 1, 1, 5, 16), [5, 3], 0, None, None, 0),
    ((3, 4, 2, 3, 20, 33), [20, 2, 0], 4, None, None, 0),
    ((2, 4, 2, 1, 9, 64), [9, 1], 1, (1, 40), None, 0),
    ((4, 4, 1, 1, 33, 72), [33, 17, 1, 0], 5, (2, 70), [70, 0], 16),
    ((6, 6, 3, 2, 40, 128), [40, 39, 2, 1, 0, 7], 16, (3, 100), [100, 1, 37], 7),
    ((4, 8, 8, 1, 64, 64), [64, 32, 31, 33], 32, (1, 129), None, 1),
    ((2, 3, 1, 40, 90, 40), [90, 20], 8, (1, 65), None, 0),       # more queries than tokens
    ((8, 16, 2, 1, 30, 32), [30] * 8, 16, (1, 300), None, 32),    # rows of a prefix in tiles
    ((2, 5, 5, 70, 200, 100), [200, 71], 64, (2, 31), [31, 31], 0),
    ((3, 2, 1, 65, 130, 192), [130, 65, 64], 128, None, None, 0),
    ((2, 2, 2, 1, 17, 256), [17, 16], 3, (1, 50), None, 10),
    ((5, 7, 1, 1, 12, 8), [12, 0, 3, 4, 5], 2, (5, 9), [9, 8, 0, 1, 2], 4),
    ((2, 1, 1, 3, 0, 16), [0, 0], 4, (1, 20), None, 0),           # a cache without room
    ((2, 2, 1, 1, 8, 24), [8, 8], 8, (1, 0), None, 0),            # a prefix without room
]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("dtype", [F32, F64])
def test_attention(hip, case, dtype):
    shape, lengths, page, prefix, prefix_lengths, prefix_page = case
    check(hip, shape, dtype, lengths, page, prefix, prefix_lengths, prefix_page)


@pytest.mark.parametrize("case", [
    ((3, 4, 1, 1, 3001, 64), [3001, 1300, 1], 16, (1, 2500), None, 0),   # both sides split
    ((3, 4, 1, 1, 1501, 40), [1501, 700, 3], 1, (3, 2047), [2047, 5, 0], 100),
    ((32, 8, 2, 1, 260, 128), [260 - 8 * i for i in range(32)], 32, (1, 1500), None, 64),
    ((24, 8, 2, 2, 100, 96), [100] * 24, 10, (2, 900), [900, 450], 33),
    ((2, 8, 2, 150, 700, 64), [700, 333], 64, (1, 600), None, 16),       # own rows in tiles
    ((2, 8, 2, 120, 500, 80), [500, 333], 12, (2, 300), None, 1),
    ((2, 4, 4, 200, 400, 66), [400, 199], 16, (1, 300), None, 0),        # odd pieces
    ((40, 12, 12, 1, 70, 160), [70 - i for i in range(40)], 1, (8, 800), [800 - 90 * i
                                                                       for i in range(8)], 128),
], ids=str)
@pytest.mark.parametrize("dtype", [F32, F64])
def test_attention_of_many_keys_and_rows(hip, case, dtype):
    shape, lengths, page, prefix, prefix_lengths, prefix_page = case
    check(hip, shape, dtype, lengths, page, prefix, prefix_lengths, prefix_page)


@pytest.mark.parametrize("gap,offset,interleaved", [(0, 0, True), (4, 4, False), (3, 1, True),
                                                    (1, 3, False)])
@pytest.mark.parametrize("queries,extent,page", [(1, 64, 16), (80, 64, 32), (80, 66, 32),
                                                 (3, 66, 5)])
def test_layouts(hip, queries, extent, page, gap, offset, interleaved):
    check(hip, (4, 8, 2, queries, 120, extent), F32, [120, 119, 81, 80], page, (2, 200),
          [200, 77], page, scale=0.3, length_type=np.int64, gap=gap, offset=offset,
          interleaved=interleaved)


def test_lengths_are_clamped_and_may_be_left_out(hip):
    b, h, hk, t, n, d = 3, 2, 1, 2, 20, 32
    query = random((b, h, t, d), F32, 1)
    cache = oracle.Pool(random((b, hk, n, d), F32, 2), random((b, hk, n, d), F32, 3), [n] * b, 5)
    shared = oracle.Pool(random((1, hk, 30, d), F32, 4), random((1, hk, 30, d), F32, 5), [30], 0)
    for lengths, prefix_lengths in (([1 << 30, -5, 7], [1 << 30]), (None, None), (None, [-1])):
        want, bound = oracle.attention(query, cache, lengths, shared, prefix_lengths)
        assert_within(attend(hip, query, cache, lengths, shared, prefix_lengths), want, bound)


@pytest.mark.parametrize("queries,heads", [(1, 2), (2, 2), (70, 4)])
@pytest.mark.parametrize("page", [5, 32])
def test_pages_that_hold_nothing(hip, queries, heads, page):
    """Tokens of pages that the cache does not have are not there: in the middle of a row, at
    its end, and all of a row's; entries of any value."""
    b, hk, n, d = 3, 2, 160, 64
    query = random((b, heads, queries, d), F32, 1)
    made = []
    for seed, rows, lengths in ((2, b, [n, n - 3, n]), (4, 1, [n])):
        pool = oracle.Pool(random((rows, hk, n, d), F32, seed), random((rows, hk, n, d), F32, 9),
                           lengths, page)
        pool.table[0, 1] = -1
        pool.table[0, 2] = len(pool.key)
        pool.table[-1, -1] = np.iinfo(np.int32).max
        pool.table[-1, 3] = np.iinfo(np.int32).min
        made.append(pool)
    made[0].table[1] = -7  # a sequence with no page at all still sees its prefix
    want, bound = oracle.attention(query, made[0], [n, n - 3, n], made[1], [n])
    got = attend(hip, query, made[0], [n, n - 3, n], made[1], [n])
    assert_within(got, want, bound)


@pytest.mark.parametrize("queries", [1, 2, 70])
@pytest.mark.parametrize("garbage", [np.nan, np.inf, np.finfo(F32).max, -np.finfo(F32).max])
@pytest.mark.parametrize("page", [0, 7, 32])
def test_what_no_query_sees_has_no_part(hip, queries, garbage, page):
    """Tokens behind a length, in the same page and in others."""
    b, h, hk, n, d = 4, 4, 2, 150, 64
    lengths, prefix_lengths = [150, 71, 70, 73], [33, 130]
    query = random((b, h, queries, d), F32, 1)
    pools = []
    for seed, rows, room, counts in ((2, b, n, lengths), (4, 2, 140, prefix_lengths)):
        pool = oracle.Pool(random((rows, hk, room, d), F32, seed),
                           random((rows, hk, room, d), F32, seed + 1), counts, page,
                           garbage=garbage)
        pools.append(pool)
    want, bound = oracle.attention(query, pools[0], lengths, pools[1], prefix_lengths)
    assert_within(attend(hip, query, pools[0], lengths, pools[1], prefix_lengths), want, bound)


@pytest.mark.parametrize("sharers,queries", [(2, 3), (40, 3)])
def test_queries_that_see_nothing_are_zero(hip, sharers, queries):
    """Queries before a sequence's first token, whatever they hold, also where what the
    others see of the prefix is not finite."""
    b, h, hk, n, d = sharers, 4, 2, 6, 64
    lengths = [i % (queries + 1) for i in range(b)]
    query = random((b, h, queries, d), F32, 1)
    for i, length in enumerate(lengths):
        query[i, :, :queries - length] = np.nan
    cache = oracle.Pool(random((b, hk, n, d), F32, 2), random((b, hk, n, d), F32, 3), lengths, 2)
    key, value = random((1, hk, 50, d), F32, 4), random((1, hk, 50, d), F32, 5)
    value[0, :, 7] = np.nan
    got = attend(hip, query, cache, lengths, oracle.Pool(key, value, [50], 0), [50])
    for i, length in enumerate(lengths):
        assert not got[i, :, :queries - length].any()
        assert np.isnan(got[i, :, queries - length:]).all()


def test_scores_of_any_size(hip):
    """Equal scores have equal weights however large they are, over both sides."""
    b, h, hk, n, d = 2, 2, 1, 40, 32
    query, key = np.ones((b, h, 1, d), F32), np.ones((b, hk, n, d), F32)
    value, prefix_value = random((b, hk, n, d), F32, 3), random((1, hk, 700, d), F32, 5)
    for size in (1.0, 1e3, 1e15, -1e3, -1e15):
        cache = oracle.Pool(key * F32(size), value, [n, n], 16)
        shared = oracle.Pool(np.full((1, hk, 700, d), F32(size)), prefix_value, [700], 16)
        got = attend(hip, query, cache, [n, n], shared, [700], scale=1.0)
        for i in range(b):
            whole = np.concatenate([prefix_value[0, 0], value[i, 0]]).astype(F64)
            # weights of 1: sums of 740 values and a product
            bound = half_step(F32) * 800 * np.abs(whole).mean(0)
            assert_within(got[i, :, 0], np.broadcast_to(whole.mean(0), (h, d)), bound)


def test_results_do_not_change_from_run_to_run(hip):
    shape = (16, 8, 2, 1, 300, 64), F32, [300 - 17 * i for i in range(16)], 16, (2, 1000), None, 16
    first = check(hip, *shape)
    for _ in range(3):
        assert np.array_equal(first, check(hip, *shape))


# ------------------------------------------------------------------- append

def turned(x, positions, freq, layout, magnitude):
    return attention_oracle.turn(x, positions, freq, layout, magnitude)


APPEND = [  # batch, heads, key heads, tokens, extent, rotary, layout, page, first place
    (1, 1, 1, 1, 1, 0, "half", 1, 0),
    (2, 4, 2, 1, 64, 64, "half", 16, 15),
    (3, 6, 2, 5, 40, 22, "half", 5, 3),
    (2, 3, 1, 7, 33, 10, "interleaved", 4, 0),
    (2, 2, 2, 9, 300, 298, "half", 3, 100),
    (4, 8, 2, 130, 128, 128, "half", 64, 1),
    (2, 5, 3, 33, 80, 32, "interleaved", 0, 2),
    (16, 9, 4, 300, 64, 64, "half", 32, 5),        # lanes that take several heads
    (16, 9, 3, 301, 128, 96, "interleaved", 7, 5),
]


@pytest.mark.parametrize("case", APPEND, ids=str)
@pytest.mark.parametrize("dtype", [F32, F64])
@pytest.mark.parametrize("place_type", [np.int32, np.int64])
def test_append(hip, case, dtype, place_type):
    """New tokens at their places, some of them padding, in caches that hold values
    already: what is not named stays as it was."""
    b, h, hk, t, d, r, layout, page, first = case
    rng = np.random.default_rng(8)
    room = first + t + 3
    pool = oracle.Pool(random((b, hk, room, d), dtype, 2), random((b, hk, room, d), dtype, 3),
                       [room] * b, page, garbage=2.5)
    cache = Cache(hip, pool, gap=3, offset=1, interleaved=bool(t % 2))
    q, k, v = (random((b, n, t, d), dtype, 10 + n) for n in (h, hk, hk))
    v = v + 1
    places = first + np.arange(t) + rng.integers(0, 4, (b, 1))
    if t > 2:
        places[:, rng.permutation(t)[:t // 3]] = -1
        places[0, 0] = room + 50  # behind the row's room
    positions = places + 1000
    freq, magnitude = attention_oracle.frequencies(r) if r else np.empty(0), 1.25
    want_key, want_value = pool.key.astype(F64), pool.value.copy()
    key_bound = np.zeros(want_key.shape)
    new, size = turned(k, positions, freq, layout, magnitude)
    for i in range(b):
        for j in range(t):
            place = places[i, j]
            if place < 0 or place >= pool.page_tokens * (1 if page == 0 else pool.table.shape[1]):
                continue
            at = (i if page == 0 else pool.table[i, place // page],
                  slice(None), place % pool.page_tokens)
            want_key[at], want_value[at] = new[i, :, j], v[i, :, j]
            key_bound[at] = attention_oracle.TURN * half_step(dtype) * size[i, :, j]
    source = [Heads(hip, x, gap=5, offset=1) for x in (q, k, v)]
    target = Heads(hip, np.zeros_like(q), gap=2)
    rotary = hip.rotary(device(hip, positions.astype(np.int64)).ptr, t, hip.INT64,
                        device(hip, freq).ptr if r else None, r, magnitude,
                        hip.ROTARY_HALF if layout == "half" else hip.ROTARY_INTERLEAVED)
    hip.call("spar_hip_launch_cache_append", cache.pages, target.heads, source[0].heads, h,
             source[1].heads, source[2].heads, b, hk, t, d,
             device(hip, places.astype(place_type)).ptr, t, hip.dtype_tag(place_type), rotary,
             hip.dtype_tag(dtype), 0)
    want, size = turned(q, positions, freq, layout, magnitude)
    assert_within(target.numpy(), want, attention_oracle.TURN * half_step(dtype) * size)
    assert not target.gaps.any()
    got_key, got_value = cache.numpy()
    assert (cache.gaps == 7).all()
    assert_within(got_key, want_key, key_bound)
    assert np.array_equal(got_value, want_value)


@pytest.mark.parametrize("tokens", [1, 40])
def test_append_in_pages_that_hold_nothing_and_without_rotation(hip, tokens):
    b, hk, d, page = 3, 2, 64, 8
    room = 48
    pool = oracle.Pool(random((b, hk, room, d), F32, 2), random((b, hk, room, d), F32, 3),
                       [room] * b, page)
    pool.table[0, 0], pool.table[0, 2] = -1, len(pool.key)
    pool.table[1] = np.iinfo(np.int32).min
    cache = Cache(hip, pool)
    k, v = random((b, hk, tokens, d), F32, 5), random((b, hk, tokens, d), F32, 6)
    places = np.broadcast_to(np.arange(tokens) + 2, (b, tokens))
    hip.call("spar_hip_launch_cache_append", cache.pages, None, None, 0, Heads(hip, k).heads,
             Heads(hip, v).heads, b, hk, tokens, d, device(hip, places[0]).ptr, 0, hip.INT64, None,
             0, 0)
    want_key, want_value = pool.key.copy(), pool.value.copy()
    for i in range(b):
        for j in range(tokens):
            number = pool.table[i, (j + 2) // page]
            if 0 <= number < len(pool.key):
                want_key[number, :, (j + 2) % page] = k[i, :, j]
                want_value[number, :, (j + 2) % page] = v[i, :, j]
    got_key, got_value = cache.numpy()
    assert np.array_equal(got_key, want_key, equal_nan=True)
    assert np.array_equal(got_value, want_value, equal_nan=True)


def test_queries_are_turned_in_place(hip):
    b, h, hk, t, d = 2, 3, 1, 4, 64
    pool = oracle.Pool(np.zeros((b, hk, 8, d), F32), np.zeros((b, hk, 8, d), F32), [8] * b, 4)
    cache = Cache(hip, pool)
    q, k = random((b, h, t, d), F32, 1), random((b, hk, t, d), F32, 2)
    query, key = Heads(hip, q), Heads(hip, k)
    freq, positions = attention_oracle.frequencies(d), np.arange(t, dtype=np.int32)
    rotary = hip.rotary(device(hip, positions).ptr, 0, hip.INT32, device(hip, freq).ptr, d)
    hip.call("spar_hip_launch_cache_append", cache.pages, query.heads, query.heads, h, key.heads,
             key.heads, b, hk, t, d, device(hip, positions).ptr, 0, hip.INT32, rotary, 0, 0)
    want, size = turned(q, positions, freq, "half", 1.0)
    assert_within(query.numpy(), want, attention_oracle.TURN * half_step(F32) * size)


def test_append_far_into_a_large_cache(hip):
    """Places whose elements are more than 2^32 from the cache's start."""
    hk, d, page, pages = 1, 128, 1 << 17, 300  # 300 * 2^24 elements of keys and of values
    count = pages * page * d
    key, value = space(hip, 4 * count), space(hip, 4 * count)
    table = device(hip, np.array([[pages - 1, 3], [pages - 2, 290]], np.int32))
    strides = (page * d, d, d)
    cache = hip.pages(key.ptr, strides, value.ptr, strides, pages, page, table.ptr, 2, 2)
    k, v = random((2, hk, 5, d), F32, 1), random((2, hk, 5, d), F32, 2)
    first = page - 2  # over the end of the first page
    places = device(hip, np.broadcast_to(first + np.arange(5), (2, 5)).astype(np.int32))
    hip.call("spar_hip_launch_cache_append", cache, None, None, 0, Heads(hip, k).heads,
             Heads(hip, v).heads, 2, hk, 5, d, places.ptr, 5, hip.INT32, None, 0, 0)
    for i in range(2):
        for j in range(5):
            number = [[pages - 1, 3], [pages - 2, 290]][i][(first + j) // page]
            at = 4 * d * (number * page + (first + j) % page)
            for buffer, x in ((key, k), (value, v)):
                got = np.empty(d, F32)
                hip.call("spar_hip_copy_device_to_host", got.ctypes.data, buffer.ptr + at, 4 * d, 0)
                assert np.array_equal(got, x[i, 0, j])
    del key, value
    _alive.clear()
    hip.call("spar_hip_empty_cache", 0)


# --------------------------------------------------------- a captured graph

def test_captured_steps_repeat_with_new_inputs(hip):
    """A token's append, attention, choice and reordering recorded into a graph: every replay
    gives what eager calls give for what the buffers hold then."""
    groups, beams, h, hk, d, n, vocabulary, prefix_tokens = 2, 3, 4, 2, 64, 40, 1003, 700
    b = groups * beams
    rng = np.random.default_rng(5)
    freq = device(hip, attention_oracle.frequencies(d))
    packed = space(hip, b * (h + 2 * hk) * d * 4)
    row = (h + 2 * hk) * d
    q, k, v = (hip.heads(packed.ptr + 4 * d * at, (row, d, row)) for at in (0, h, h + hk))
    places, positions = space(hip, 8 * b), space(hip, 8 * b)
    lengths, logits, scores = space(hip, 4 * b), space(hip, 4 * b * vocabulary), space(hip, 4 * b)
    table = device(hip, rng.permutation(b * n).reshape(b, n).astype(np.int32))
    prefix = [device(hip, random((groups, hk, prefix_tokens, d), F32, 3 + i)) for i in range(2)]
    shared = hip.pages(prefix[0].ptr, (hk * prefix_tokens * d, prefix_tokens * d, d),
                       prefix[1].ptr, (hk * prefix_tokens * d, prefix_tokens * d, d), groups,
                       prefix_tokens)
    rotary = hip.rotary(positions.ptr, 1, hip.INT64, freq.ptr, d)
    shape = hip.cache_attention(b, groups, h, hk, 1, d, 0.125, lengths.ptr, None, hip.INT32, 0)
    choice = hip.beams(groups, beams, vocabulary, beams, vocabulary, None, -1, 0)

    def buffers():
        made = {name: device(hip, np.zeros(b * n * hk * d, F32)) for name in ("key", "value")}
        made |= {name: space(hip, b * h * d * 4) for name in ("turned", "output")}
        made |= {"scores": space(hip, 4 * b), "parents": space(hip, 8 * b),
                 "tokens": space(hip, 8 * b), "table": space(hip, 4 * b * n)}
        made["pages"] = hip.pages(made["key"].ptr, (hk * d, d, d), made["value"].ptr,
                                  (hk * d, d, d), b * n, 1, table.ptr, n, n)
        made["need"] = (hip.cache_attention_workspace(made["pages"], shared, shape),
                        hip.beam_select_workspace(choice))
        made["work"] = [space(hip, size) for size in made["need"]]
        return made

    def run(m):
        turned_heads = hip.heads(m["turned"].ptr, (h * d, d, h * d))
        hip.call("spar_hip_launch_cache_append", m["pages"], turned_heads, q, h, k, v, b, hk, 1, d,
                 places.ptr, 1, hip.INT64, rotary, 0, 0)
        hip.call("spar_hip_launch_cache_attention", hip.heads(m["output"].ptr, (h * d, d, h * d)),
                 turned_heads, m["pages"], shared, shape, m["work"][0].ptr, m["need"][0], 0)
        hip.call("spar_hip_launch_beam_select", m["scores"].ptr, m["parents"].ptr,
                 m["tokens"].ptr, None, logits.ptr, scores.ptr, choice, m["work"][1].ptr,
                 m["need"][1], 0)
        hip.call("spar_hip_launch_reorder", hip.reorders((m["table"].ptr, n, table.ptr, n, n, 4)),
                 1, m["parents"].ptr, b, b, 0)

    def put(buffer, values):
        values = np.ascontiguousarray(values)
        hip.call("spar_hip_copy_host_to_device", buffer.ptr, values.ctypes.data, values.nbytes, 0)

    def refill(seed):
        rng = np.random.default_rng(seed)
        put(packed, rng.standard_normal((b, row)).astype(F32))
        put(logits, 3 * rng.standard_normal((b, vocabulary)).astype(F32))
        put(scores, rng.standard_normal(b).astype(F32))
        put(places, np.full(b, seed, np.int64))
        put(positions, np.full(b, seed + prefix_tokens, np.int64))
        put(lengths, np.full(b, seed + 1, np.int32))

    captured, eager = buffers(), buffers()
    refill(0)
    run(captured)
    run(eager)
    hip.synchronize()
    lib = ctypes.CDLL("libamdhip64.so")
    stream, graph, executable = (ctypes.c_void_p() for _ in range(3))
    hip.call("spar_hip_stream", ctypes.byref(stream), 0)
    assert lib.hipStreamBeginCapture(stream, 2) == 0
    run(captured)
    assert lib.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert lib.hipGraphInstantiate(ctypes.byref(executable), graph, None, None, 0) == 0
    for seed in (1, 2, 3, 4):
        refill(seed)
        run(eager)
        assert lib.hipGraphLaunch(executable, stream) == 0
        hip.synchronize()
        for name, kind, count in (("key", F32, b * n * hk * d), ("output", F32, b * h * d),
                                  ("scores", F32, b), ("parents", np.int64, b),
                                  ("tokens", np.int64, b), ("table", np.int32, b * n)):
            assert np.array_equal(captured[name].to_numpy(kind, (count,)),
                                  eager[name].to_numpy(kind, (count,))), (seed, name)
    lib.hipGraphExecDestroy(executable)
    lib.hipGraphDestroy(graph)
