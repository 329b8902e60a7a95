"""How large a call of attention over caches may be: what its launches cannot count is
refused on the host, before any device call, and nothing else is."""
import ctypes

import pytest

from spar_amd import hip

A = 1 << 20  # an address that is never read
NO_DEVICE = 999  # calls that pass the checks end here
GROUPS = (1 << 24) - 1  # workgroups of a launch


def pages(page_tokens=16, table_pages=4):
    return hip.pages(A, (64, 64, 64), A, (64, 64, 64), 8, page_tokens, A, 4, table_pages)


def attend(batch, heads, key_heads, queries, prefixes=0, room=4):
    """(whether the call passes, bytes of its workspace)."""
    cache, prefix = pages(table_pages=room), pages() if prefixes else None
    call = hip.cache_attention(batch, prefixes, heads, key_heads, queries, 64, 1.0, A,
                               A if prefixes else None, hip.INT32, 0)
    need = ctypes.c_uint64(0)
    status = hip.status_of("spar_hip_cache_attention_workspace", ctypes.byref(need), cache, prefix,
                           call).code
    heads_of = hip.heads(A, (64, 64, 64))
    done = hip.status_of("spar_hip_launch_cache_attention", heads_of, heads_of, cache, prefix,
                         call, A, need.value, NO_DEVICE).code
    assert (status == 0) == (done != 1)  # the two agree
    return done not in (0, 1), need.value


@pytest.mark.parametrize("batch,heads,queries", [
    (64, 32, 8191), (64, 32, 8192), (4, 32, 131072), (1, 32, 524288), (1, 32, (1 << 25) - 17)])
@pytest.mark.parametrize("room", [0, 4])
def test_rows_without_a_prefix_need_no_join(batch, heads, queries, room):
    assert attend(batch, heads, 8, queries, room=room) == (True, 0)


@pytest.mark.parametrize("prefixes", [1, 2])
def test_rows_behind_a_prefix_are_as_many_as_a_join_takes(prefixes):
    # two parts: eight rows a workgroup of the join
    most = 8 * GROUPS
    assert most == 32 * (1 << 22) - 8
    for batch, queries, passes in ((8, 1 << 17, True), (32, (1 << 17) - 1, True),
                                   (32, 1 << 17, False), (64, 1 << 17, False)):
        taken, need = attend(batch, 32, 8, queries, prefixes)
        rows = batch * 32 * queries
        assert taken == passes == (rows <= most)
        assert need == (2 * rows * (64 + 2) * 4 if passes else 0)
    # to the row: 16 sequences of 8 heads with the last query that fits, and one more
    queries = most // (16 * 8)
    assert 16 * 8 * queries <= most < 16 * 8 * (queries + 1)
    assert attend(16, 8, 8, queries, prefixes)[0]
    assert not attend(16, 8, 8, queries + 1, prefixes)[0]


def test_workgroups_are_as_many_as_a_launch_counts():
    # 64 rows each, of one key head of a sequence
    assert attend(1 << 16, 8, 8, 32 * 64 - 65)[0]      # 31 tiles of 2^19 key heads
    assert not attend(1 << 16, 8, 8, 32 * 64)[0]       # 2^24
    assert attend(GROUPS, 1, 1, 1)[0]
    assert not attend(GROUPS + 1, 1, 1, 1)[0]
    # both sides together: the prefixes' tiles of 64 rows and the sequences' groups
    assert attend((1 << 20) - 1, 8, 8, 1, (1 << 20) - 1)[0]  # 2^23 - 8 of either
    assert not attend(1 << 20, 8, 8, 1, 1 << 20)[0]
