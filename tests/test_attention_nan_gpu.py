"""How far a NaN or an infinity in an input of attention reaches in its gradients: those of
its key head and of the query heads that read it, and no others."""
import numpy as np
import pytest

from tests.test_attention_gpu import F32, F64, _release_buffers, attend, inputs  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("where", ["query", "key", "value", "gradient"])
@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("batch,tokens,dtype", [(2, 40, F32), (2, 40, F64),
                                                (60, 100, F32), (60, 100, F64),  # in tiles
                                                (2, 900, F32)])                  # in parts
def test_gradients_of_other_heads_and_sequences_stay(hip, where, value, batch, tokens, dtype):
    arrays = dict(zip(("query", "key", "value", "gradient"),
                      inputs(batch, 4, 2, tokens, tokens, 64, dtype)))

    def run():
        return attend(hip, arrays["query"], arrays["key"], arrays["value"], 10, 2,
                      gradient=arrays["gradient"], out_fill=7.0)

    output, _, gradients = run()
    # in the first sequence's second key head, which its last two query heads read
    arrays[where][0, 1 if where in ("key", "value") else 2, 20, 5] = value
    marked, _, made = run()
    for clean, x, group in zip((output, *gradients), (marked, *made), (2, 2, 1, 1)):
        assert np.array_equal(clean[1:], x[1:])
        assert np.array_equal(clean[0, :group], x[0, :group])
    dq, dk, dv = made
    assert not np.isfinite(dq[0, 2, 20]).all()
    if where in ("key", "value", "query"):
        assert not np.isfinite(dk[0, 1]).all()


@pytest.mark.parametrize("garbage", [np.nan, np.inf, np.finfo(F32).max])
@pytest.mark.parametrize("batch,tokens", [(2, 40), (60, 100)])
def test_gradients_beside_what_no_query_sees(hip, garbage, batch, tokens):
    """Keys and values behind a sequence's length, and queries and gradients in front of
    it: the same bits as with other numbers there."""
    q, k, v, g = inputs(batch, 4, 2, tokens, tokens, 64, F32)
    lengths = np.full(batch, tokens, np.int32)
    lengths[::2] = tokens - 17
    runs = []
    for fill in (garbage, 1.0):
        for x in (k, v):
            x[::2, :, tokens - 17:] = fill
        for x in (q, g):
            x[::2, :, :17] = fill
        runs.append(attend(hip, q, k, v, 10, 2, lengths=lengths, gradient=g, out_fill=7.0))
    for x, y in zip((runs[0][0], *runs[0][2]), (runs[1][0], *runs[1][2])):
        assert np.array_equal(x, y)
        assert np.isfinite(x).all()
