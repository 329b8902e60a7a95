"""Beam search whose own tokens lie in pages of several: picks that go on from one parent get
pages of their own, with a copy of what the shared one holds, before they are appended to."""
import numpy as np
import pytest

from tests import attention_oracle
from tests.test_decoding_api_gpu import Model, get, put, search, sp  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def own_pages(sp, cache, table, place):
    """Gives every row of a table that has been put in the order of its parents a page of its
    own for its token `place`; tokens before it in the page are copied.  Returns the table."""
    rows = get(sp, table).copy()
    page_tokens = cache.key.shape[2]
    entry, slot = place // page_tokens, place % page_tokens
    shared = rows[:, entry].astype(np.int64)
    named = rows[:, :entry + (slot != 0)]
    fresh = np.setdiff1d(np.arange(cache.key.shape[0], dtype=np.int32), named)[:len(rows)]
    assert len(fresh) == len(rows)
    rows[:, entry], rows[:, entry + 1:] = fresh, -1
    kept = sp.reorder([cache.key, cache.value], put(sp, shared)) if slot else None
    cache.table = put(sp, rows)
    if kept:
        at = np.arange(page_tokens)
        places = np.where(at < slot, entry * page_tokens + at, -1)
        sp.cache_append(cache, *kept, put(sp, np.broadcast_to(places, (len(rows), page_tokens))))
    return cache.table


@pytest.mark.parametrize("page", [2, 3, 16])
def test_beams_of_one_parent(sp, page):  # noqa: F811
    """Two prompts of one length, four beams each; the definition keeps all tokens of every
    beam.  In double: totals of both differ by rounding alone (scores of about 10 over 20 keys,
    sums of 12 products: some 10^4 u = 1e-12); 1e-10 leaves 100 times that, and the best totals
    are checked to lie further apart."""
    model = Model(4, 2, 12, 50)
    rng = np.random.default_rng(41)
    prompts = [rng.integers(0, 50, 7) for _ in range(2)]
    groups, beams, steps, end = 2, 4, 8, 30
    want = search(model, prompts, beams, steps, end)
    rows = groups * beams
    h, hk, d = model.heads, model.key_heads, model.extent
    freq = put(sp, model.freq)
    entries = -(-steps // page)
    count = rows * (entries + 1)
    cache = sp.PagedCache(put(sp, np.full((count, hk, page, d), np.nan)),
                          put(sp, np.full((count, hk, page, d), np.nan)))
    table = np.full((rows, entries), -1, np.int32)
    table[:, 0] = rng.permutation(count)[:rows]
    cache.table = put(sp, table)
    known = len(prompts[0]) - 1
    q, k, v = (put(sp, x).transpose(1, 2) for x in model.split(np.array(prompts)[:, :-1]))
    prefix = sp.PagedCache(put(sp, np.zeros((groups, hk, known, d))),
                           put(sp, np.zeros((groups, hk, known, d))))
    at = np.broadcast_to(np.arange(known), (groups, known))
    sp.cache_append(prefix, k, v, put(sp, at), sp.CacheRotation(put(sp, at), freq))

    tokens = np.repeat([p[-1] for p in prompts], beams)
    scores = np.full((groups, beams), -np.inf)
    scores[:, 0] = 0
    scores, ended = put(sp, scores), put(sp, np.zeros((groups, beams), np.int32))
    made = np.zeros((rows, 0), np.int64)
    twins = 0
    for step in range(steps):
        q, k, v = (put(sp, x[:, None]).transpose(1, 2) for x in model.split(tokens))
        positions = put(sp, np.full((rows, 1), known + step))
        query = sp.cache_append(cache, k, v, put(sp, np.full((rows, 1), step)),
                                sp.CacheRotation(positions, freq), q)
        out = sp.cache_attention(query, cache, put(sp, np.full(rows, step + 1, np.int32)), prefix)
        x = get(sp, out).transpose(0, 2, 1, 3).reshape(rows, h * d) @ model.output
        picked = sp.beam_select(put(sp, x.reshape(groups, beams, -1)), scores, beams, end, ended)
        scores, ended = picked.scores, picked.ended
        parents, tokens = get(sp, picked.parents).ravel(), get(sp, picked.tokens).ravel()
        made = np.concatenate([made[parents], tokens[:, None]], 1)
        if step + 1 < steps:
            [table] = sp.reorder([cache.table], picked.parents)
            own_pages(sp, cache, table, step + 1)
            twins += (step + 1) % page != 0 and len(np.unique(parents)) < rows
    assert twins > 1  # pages in the middle of which two picks had one parent
    totals, flags = get(sp, scores), get(sp, ended)
    for i in range(groups):
        best = [s["score"] for s in want[i]]
        assert min(a - b for a, b in zip(best, best[1:])) > 1e-8
        for j, state in enumerate(want[i]):
            assert made[i * beams + j].tolist() == state["made"]
            assert abs(totals[i, j] - state["score"]) <= 1e-10 * abs(state["score"])
            assert flags[i, j] == state["ended"]
