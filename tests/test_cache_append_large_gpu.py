"""Appends of whole float32 halves that write more than 64 MiB, whose stores go past the
caches, against the definition."""
import numpy as np
import pytest

from tests import test_cache_attention_gpu as attention
from tests.test_cache_attention_gpu import _release_buffers  # noqa: F401  (releases buffers)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", [  # batch, heads, key heads, tokens, extent, rotary, layout, page,
    (3, 9, 3, 5900, 64, 64, "half", 32, 5),     # first place
    (2, 5, 3, 6001, 128, 128, "half", 7, 1),
    (2, 6, 2, 6600, 128, 128, "half", 0, 0),
], ids=str)
@pytest.mark.parametrize("place_type", [np.int32, np.int64])
def test_append_past_the_caches(hip, case, place_type):
    """Odd and even numbers of heads, padding, ends of pages and of the rows' room, values that
    stay between."""
    batch, heads, key_heads, tokens, extent = case[:5]
    assert batch * tokens * (heads + 2 * key_heads) * extent * 4 >= 64 << 20
    assert extent // 2 * 4 % 128 == 0
    attention.test_append(hip, case, np.float32, place_type)
