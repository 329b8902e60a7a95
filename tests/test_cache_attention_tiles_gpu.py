"""Attention over caches where rows fill tiles, where a workgroup reads many pages, and where
few rows share a prefix: every way the kernels go, against the definition in 64 bits."""
import numpy as np
import pytest

from tests import decoding_oracle as oracle
from tests.attention_oracle import assert_within
from tests.test_cache_attention_gpu import (  # noqa: F401  (the fixture releases buffers)
    F32, F64, _release_buffers, attend, check, random)

pytestmark = pytest.mark.gpu


def fills_tiles(rows, units, room):
    """Whether tiles of 64 rows are taken: more than 32 rows, and tiles for the chip."""
    return rows > 32 and -(-rows // 64) * units * max(1, room // 256) >= 192


# (batch, heads, key heads, queries, room, extent), lengths, page, prefix (rows, room), page
PREFIXES = [
    ((64, 64, 8, 1, 40, 128), 16, (8, 800), 16),      # single tokens, whole pages
    ((64, 64, 8, 1, 40, 128), 5, (8, 800), 7),        # and pages that end inside tiles
    ((64, 64, 8, 1, 33, 64), 1, (8, 777), 32),
    ((64, 64, 8, 1, 21, 96), 8, (8, 800), 0),
    ((64, 64, 8, 1, 21, 40), 32, (8, 771), 64),
    ((64, 64, 8, 1, 30, 66), 16, (8, 800), 16),       # pieces that do not divide a head
    ((32, 128, 8, 1, 30, 256), 16, (4, 1600), 64),    # sixteen rows of a sequence
    ((32, 128, 8, 1, 30, 192), 3, (4, 1600), 1),
    ((40, 40, 8, 2, 30, 32), 16, (8, 800), 100),      # more rows than a tile
]


@pytest.mark.parametrize("case", PREFIXES, ids=str)
@pytest.mark.parametrize("dtype", [F32, F64])
def test_prefixes_in_tiles(hip, case, dtype):
    shape, page, (rows, room), prefix_page = case
    b, h, hk, t, n, _ = shape
    assert fills_tiles(b // rows * t * h // hk, rows * hk, room)
    lengths = [n - n * i // b for i in range(b)]
    counts = [room - (room - 1) * i // rows for i in range(rows)]
    check(hip, shape, dtype, lengths, page, (rows, room), counts, prefix_page)


@pytest.mark.parametrize("page,prefix_page", [(16, 16), (7, 0), (0, 48)])
@pytest.mark.parametrize("extent", [64, 72, 100, 130])
@pytest.mark.parametrize("dtype", [F32, F64])
def test_queries_in_tiles(hip, extent, page, prefix_page, dtype):
    """Both sides in tiles: many queries of many sequences, some before the first token."""
    b, h, hk, t, n = 24, 16, 8, 40, 70
    assert fills_tiles(t * h // hk, b * hk, n) and fills_tiles(b // 3 * t * h // hk, 3 * hk, 90)
    lengths = [n - n * i // (b - 1) for i in range(b)]
    check(hip, (b, h, hk, t, n, extent), dtype, lengths, page, (3, 600), [600, 0, 301], prefix_page)


@pytest.mark.parametrize("page", [5, 16, 64])
def test_tiles_of_pages_that_hold_nothing(hip, page):
    """In the middle of a prefix, at its start and its end, and all of a prefix."""
    b, h, hk, n, d, rows, room = 64, 64, 8, 20, 128, 8, 800
    query = random((b, h, 1, d), F32, 1)
    cache = oracle.Pool(random((b, hk, n, d), F32, 2), random((b, hk, n, d), F32, 3), [n] * b, 4)
    prefix = oracle.Pool(random((rows, hk, room, d), F32, 4), random((rows, hk, room, d), F32, 5),
                         [room] * rows, page)
    prefix.table[0, 0] = prefix.table[1, 3] = prefix.table[1, 4] = -1
    prefix.table[2, -1] = len(prefix.key)
    prefix.table[3] = np.iinfo(np.int32).min
    prefix.table[4, ::2] = np.iinfo(np.int32).max
    want, bound = oracle.attention(query, cache, [n] * b, prefix, [room] * rows)
    assert_within(attend(hip, query, cache, [n] * b, prefix, [room] * rows), want, bound)


@pytest.mark.parametrize("interleaved,gap,offset", [(True, 0, 0), (False, 4, 4), (False, 1, 3)])
def test_layouts_in_tiles(hip, interleaved, gap, offset):
    check(hip, (64, 64, 8, 1, 24, 64), F32, [24 - i % 5 for i in range(64)], 8, (8, 800),
          [800 - i for i in range(8)], 32, interleaved=interleaved, gap=gap, offset=offset)


def test_queries_before_the_first_token_in_tiles(hip):
    """Zeros, whatever they hold and whatever others see of their prefix."""
    b, h, hk, t, n, d = 64, 64, 8, 1, 4, 64
    lengths = [i % 2 * 3 for i in range(b)]
    query = random((b, h, t, d), F32, 1)
    query[::2] = np.nan
    cache = oracle.Pool(random((b, hk, n, d), F32, 2), random((b, hk, n, d), F32, 3), lengths, 2)
    key, value = random((8, hk, 800, d), F32, 4), random((8, hk, 800, d), F32, 5)
    value[:, :, 7] = np.nan
    got = attend(hip, query, cache, lengths, oracle.Pool(key, value, [800] * 8, 16), None)
    assert not got[::2].any() and np.isnan(got[1::2]).all()


@pytest.mark.parametrize("extent,dtype", [(16, F32), (16, F64), (72, F32)])
@pytest.mark.parametrize("heads", [8, 48])
def test_more_pages_than_a_wave_has_lanes(hip, extent, dtype, heads):
    """So many sequences that one workgroup reads all pages of a row, at most 82."""
    b, hk, n = 96, 8, 1300
    lengths = [n - 13 * i for i in range(b)]
    check(hip, (b, heads, hk, 1, n, extent), dtype, lengths, 16)


@pytest.mark.parametrize("heads,key_heads", [(1, 1), (3, 1), (4, 1), (4, 2)])
@pytest.mark.parametrize("extent", [1, 6, 32, 64, 65, 100, 128, 192, 256])
def test_few_rows(hip, heads, key_heads, extent):
    """A prefix of one sequence each, so that neither side has more than four rows."""
    lengths = [90, 17, 0, 1, 8]
    check(hip, (5, heads, key_heads, 1, 90, extent), F32, lengths, 4, (5, 150), [150, 9, 3, 0, 16],
          16)
    check(hip, (5, heads, key_heads, 1, 90, extent), F32, lengths, 16, (5, 150), [150, 9, 3, 0, 16],
          9, gap=1, offset=1)
