"""The decoding operators through the tensor API: beam search behind shared prompts from
the prompt to the last token, views and refusals."""
import numpy as np
import pytest

from tests import attention_oracle, decoding_oracle as oracle
from tests.attention_oracle import assert_within

pytestmark = pytest.mark.gpu

F32, F64 = np.float32, np.float64


@pytest.fixture(scope="module")
def sp():
    from spar_amd import spar

    if spar.hip_device_count() < 1:
        pytest.fail("no HIP device visible to a gpu-marked test")
    return spar


def put(sp, array):
    return sp.Tensor.from_numpy(np.ascontiguousarray(array)).to(sp.Device.hip(0))


def get(sp, tensor):
    return tensor.contiguous().to(sp.Device.cpu()).numpy()


class Model:
    """One layer of attention over embedded tokens, the same for device and definition."""

    def __init__(self, heads, key_heads, extent, vocabulary):
        rng = np.random.default_rng(31)
        self.heads, self.key_heads, self.extent = heads, key_heads, extent
        self.packed = rng.standard_normal((vocabulary, (heads + 2 * key_heads) * extent))
        self.output = rng.standard_normal((heads * extent, vocabulary)) * 0.3
        self.freq = attention_oracle.frequencies(extent)

    def split(self, tokens):
        """[..., heads, extent] queries, keys and values of tokens."""
        every = self.packed[tokens].reshape(*tokens.shape, -1, self.extent)
        h, hk = self.heads, self.key_heads
        return every[..., :h, :], every[..., h:h + hk, :], every[..., h + hk:, :]


def turned(x, position, freq):
    """x [heads, extent] turned by one position."""
    return attention_oracle.turn(x[None, :, None], np.array([position]), freq, "half")[0][0, :, 0]


def search(model, prompts, beams, steps, end):
    """Beam search by its definition: every beam keeps its tokens and all its keys and values."""
    g = model.heads // model.key_heads
    found = []
    for prompt in prompts:
        states = []
        for i in range(beams):
            states.append(dict(score=0.0 if i == 0 else -np.inf, tokens=list(prompt), ended=False,
                               made=[]))
        for step in range(steps):
            totals = []
            for i, state in enumerate(states):
                q, k, v = model.split(np.array(state["tokens"]))
                n = len(state["tokens"])
                keys = np.stack([turned(k[t], t, model.freq) for t in range(n)])
                query = turned(q[-1], n - 1, model.freq)
                out = []
                for h in range(model.heads):
                    scores = keys[:, h // g] @ query[h] / np.sqrt(model.extent)
                    weights = np.exp(scores - scores.max())
                    out.append(weights / weights.sum() @ v[:, h // g])
                x = np.concatenate(out) @ model.output
                logits = x - (x.max() + np.log(np.exp(x - x.max()).sum()))
                if state["ended"]:
                    logits = np.where(np.arange(len(x)) == end, 0.0, -np.inf)
                totals += [(-(state["score"] + y), i, t) for t, y in enumerate(logits)]
            best = sorted(totals)[:beams]
            states = [dict(score=-total, tokens=states[i]["tokens"] + [t],
                           made=states[i]["made"] + [t], ended=states[i]["ended"] or t == end)
                      for total, i, t in best]
        found.append(states)
    return found


@pytest.mark.parametrize("page", [1, 0])
@pytest.mark.parametrize("prefix_page", [4, 0])
def test_beam_search(sp, page, prefix_page):
    """Two prompts of different lengths, three beams each: the prompts' keys and values are
    kept once, the beams' own tokens in pages of one token, whose tables move with their beams,
    or in a contiguous cache, whose rows do.

    In double: totals of both differ by rounding alone (scores of about 10 over 20 keys, sums
    of 12 products: some 10^4 u = 1e-12); 1e-10 leaves 100 times that, and the best totals are
    checked to lie further apart."""
    model = Model(4, 2, 12, 50)
    rng = np.random.default_rng(32)
    prompts = [rng.integers(0, 50, n) for n in (11, 6)]
    beams, steps, end, groups = 3, 6, 30, 2
    want = search(model, prompts, beams, steps, end)
    rows, room = groups * beams, steps + 1
    h, hk, d = model.heads, model.key_heads, model.extent
    freq = put(sp, model.freq)

    def cache_of(count, tokens, size):
        if size == 0:
            return sp.PagedCache(put(sp, np.full((count, hk, tokens, d), np.nan)),
                                 put(sp, np.full((count, hk, tokens, d), np.nan)))
        entries = -(-tokens // size)
        pages = rng.permutation(count * entries).reshape(count, entries)
        return sp.PagedCache(put(sp, np.full((pages.size, hk, size, d), np.nan)),
                             put(sp, np.full((pages.size, hk, size, d), np.nan)),
                             put(sp, pages.astype(np.int32)))

    # all but the prompts' last tokens, padded in front, into the prefixes' rows
    longest = max(len(p) for p in prompts) - 1
    prefix = cache_of(groups, longest, prefix_page)
    padded = np.zeros((groups, longest), np.int64)
    places = np.full((groups, longest), -1)
    for i, prompt in enumerate(prompts):
        n = len(prompt) - 1
        padded[i, longest - n:], places[i, longest - n:] = prompt[:-1], np.arange(n)
    q, k, v = (put(sp, x).transpose(1, 2) for x in model.split(padded))
    sp.cache_append(prefix, k, v, put(sp, places),
                    sp.CacheRotation(put(sp, np.maximum(places, 0)), freq))
    prefix_lengths = np.array([len(p) - 1 for p in prompts], np.int32)

    cache = cache_of(rows, room, page)
    tokens = np.repeat([p[-1] for p in prompts], beams)
    scores = np.full((groups, beams), -np.inf)
    scores[:, 0] = 0
    scores, ended = put(sp, scores), put(sp, np.zeros((groups, beams), np.int32))
    history = put(sp, np.full((rows, steps), -1, np.int64))
    starts = np.repeat(prefix_lengths, beams)[:, None].astype(np.int64)
    for step in range(steps):
        q, k, v = (put(sp, x[:, None]).transpose(1, 2) for x in model.split(tokens))
        query = sp.cache_append(cache, k, v, put(sp, np.full((rows, 1), step, np.int32)),
                                sp.CacheRotation(put(sp, starts + step), freq), q)
        out = sp.cache_attention(query, cache, put(sp, np.full(rows, step + 1, np.int32)), prefix,
                                 put(sp, prefix_lengths))
        x = get(sp, out).transpose(0, 2, 1, 3).reshape(rows, h * d) @ model.output
        picked = sp.beam_select(put(sp, x.reshape(groups, beams, -1)), scores, beams, end, ended)
        scores, ended = picked.scores, picked.ended
        if page:
            table, history = sp.reorder([cache.table, history], picked.parents)
            # pages that beams share so far are full; new tokens come into new ones
            fresh = get(sp, table).copy()
            unused = np.setdiff1d(np.arange(cache.key.shape[0]), fresh[:, :step + 1])
            fresh[:, step + 1:] = -1
            fresh[:, step + 1] = unused[:rows]
            cache.table = put(sp, fresh)
        else:
            cache.key, cache.value, history = sp.reorder([cache.key, cache.value, history],
                                                         picked.parents)
        tokens = get(sp, picked.tokens).ravel()
        made = get(sp, history).copy()
        made[:, step] = tokens
        history = put(sp, made)
    totals, flags = get(sp, scores), get(sp, ended)
    for i in range(groups):
        best = [s["score"] for s in want[i]]
        assert min(a - b for a, b in zip(best, best[1:])) > 1e-8
        for j, state in enumerate(want[i]):
            assert get(sp, history)[i * beams + j].tolist() == state["made"]
            assert abs(totals[i, j] - state["score"]) <= 1e-10 * abs(state["score"])
            assert flags[i, j] == state["ended"]


def random(shape, dtype, seed):
    return np.random.default_rng(seed).standard_normal(shape).astype(dtype)


def test_views_are_read_and_written_in_place(sp):
    """A layer's part of a cache of several layers, keys and values side by side, tables and
    lengths that are columns of others, heads of a packed projection."""
    b, h, hk, d, page, n = 3, 4, 2, 32, 8, 30
    layers = put(sp, np.zeros((12, page, 3, 2, hk, d), F32))  # page, token, layer, k and v
    table = np.random.default_rng(1).permutation(12).reshape(3, 4).astype(np.int32)
    key, value = (layers.reshape([12, page, 6 * hk, d]).transpose(1, 2).narrow(1, at * hk, hk)
                  for at in (2, 3))
    columns = put(sp, np.concatenate([table + 100, table, table + 200], 1)).narrow(1, 4, 4)
    cache = sp.PagedCache(key, value, columns)
    packed = random((b, n, (h + 2 * hk) * d), F32, 2)
    every = put(sp, packed).reshape([b, n, h + 2 * hk, d]).transpose(1, 2)
    places = np.broadcast_to(np.arange(n), (b, n))
    freq = attention_oracle.frequencies(d)
    turned = sp.cache_append(cache, every.narrow(1, h, hk), every.narrow(1, h + hk, hk),
                             put(sp, places),
                             sp.CacheRotation(put(sp, np.arange(n)), put(sp, freq)),
                             every.narrow(1, 0, h))
    heads = packed.reshape(b, n, h + 2 * hk, d).swapaxes(1, 2)
    want, size = attention_oracle.turn(heads[:, :h + hk], np.arange(n), freq, "half")
    bound = attention_oracle.TURN * attention_oracle.half_step(F32) * size
    assert_within(get(sp, turned), want[:, :h], bound[:, :h])
    stored = get(sp, layers)
    for i in range(b):
        for t in range(n):
            at = stored[table[i, t // page], t % page]
            assert_within(at[1, 0], want[i, h:, t], bound[i, h:, t])
            assert np.array_equal(at[1, 1], heads[i, h + hk:, t])
            assert not at[0].any() and not at[2].any()
    pool = oracle.Pool(np.zeros((b, hk, n, d), F32), np.zeros((b, hk, n, d), F32), [n] * b, page)
    pool.table = table
    pool.key = stored[:, :, 1, 0].swapaxes(1, 2)
    pool.value = stored[:, :, 1, 1].swapaxes(1, 2)
    query = get(sp, turned)
    want, bound = oracle.attention(query, pool, [n, 9, n])
    got = sp.cache_attention(turned, cache, put(sp, np.array([n, 9, n])))
    assert_within(get(sp, got), want, bound)


def test_logits_of_views(sp):
    whole = 3 * random((2, 3, 2, 900), F32, 3)
    scores = random((3, 2), F32, 4)
    x, s = put(sp, whole), put(sp, scores)
    six = x.reshape([2, 6, 900])
    for view, values, before in (
            (x.narrow(0, 1, 1).reshape([3, 2, 900]), whole[1], scores),
            (six.narrow(2, 5, 700), whole.reshape(2, 6, 900)[..., 5:705], None),
            (six.narrow(1, 1, 3), whole.reshape(2, 6, 900)[:, 1:4], None),
            (six.transpose(0, 1), whole.reshape(2, 6, 900).swapaxes(0, 1), None),
            (six.narrow(2, 0, 30).transpose(1, 2), whole.reshape(2, 6, 900)[..., :30].swapaxes(1, 2),
             None)):
        given = s if before is not None else put(sp, np.zeros(values.shape[:2], F32))
        picked = sp.beam_select(view, given, 4)
        want = oracle.select(values, np.zeros(values.shape[:2]) if before is None else before, 4)
        assert oracle.border(values, get(sp, given), 4) > 2 * oracle.select_bound(values, F32)
        assert np.array_equal(get(sp, picked.parents), want[1])
        assert np.array_equal(get(sp, picked.tokens), want[2])
        assert not get(sp, picked.ended).any()


def test_reorder_of_views_and_no_states(sp):
    x = np.arange(60.0).reshape(5, 4, 3)
    parents = put(sp, np.array([[4, 0], [0, 9]]))
    made = sp.reorder([put(sp, x).transpose(1, 2), put(sp, np.arange(5, dtype=np.int32))], parents)
    order = np.array([4, 0, 0])
    assert np.array_equal(get(sp, made[0])[:3], x.swapaxes(1, 2)[order])
    assert not get(sp, made[0])[3].any()
    assert get(sp, made[1]).tolist() == [4, 0, 0, 0]
    assert sp.reorder([], parents) == []


def test_calls_of_nothing(sp):
    none = put(sp, np.zeros((0, 2, 1, 8), F32))
    cache = sp.PagedCache(put(sp, np.zeros((4, 2, 4, 8), F32)), put(sp, np.zeros((4, 2, 4, 8), F32)),
                          put(sp, np.zeros((0, 3), np.int32)))
    assert sp.cache_append(cache, none, none, put(sp, np.zeros((0, 1), np.int32))) is None
    assert tuple(sp.cache_attention(none, cache).shape) == (0, 2, 1, 8)
    picked = sp.beam_select(put(sp, np.zeros((0, 2, 5), F32)), put(sp, np.zeros((0, 2), F32)), 3)
    assert tuple(picked.tokens.shape) == (0, 3)


def test_refusals(sp):
    b, h, hk, t, d, page = 4, 4, 2, 1, 16, 4
    x = put(sp, np.zeros((b, h, t, d), F32))
    k = put(sp, np.zeros((b, hk, t, d), F32))
    pool = put(sp, np.zeros((9, hk, page, d), F32))
    table = put(sp, np.zeros((b, 3), np.int32))
    cache = sp.PagedCache(pool, pool, table)
    places = put(sp, np.zeros((b, t), np.int64))
    rotation = sp.CacheRotation(places, put(sp, attention_oracle.frequencies(d)))

    def refused(match, call, *args, **options):
        with pytest.raises(ValueError, match=match):
            call(*args, **options)

    wide = put(sp, np.zeros((b, hk, t, 2 * d), F32))
    double = put(sp, np.zeros((b, hk, t, d), F64))
    tracked = put(sp, np.zeros((b, hk, t, d), F32))
    tracked.set_requires_grad(True)
    other = put(sp, np.zeros((9, hk, 2 * page, d), F32))
    refused("extents differ", sp.cache_append, cache, wide, wide, places)
    refused("one dtype", sp.cache_append, cache, double, double, places)
    refused("one shape", sp.cache_append, cache, k, wide, places)
    refused("detach", sp.cache_append, cache, tracked, k, places)
    refused("one shape", sp.cache_append, sp.PagedCache(pool, other, table), k, k, places)
    refused("row for every", sp.cache_append, sp.PagedCache(pool, pool), k, k, places)
    refused("heads differ", sp.cache_append, cache, x, x, places)
    refused("rotation", sp.cache_append, cache, k, k, places, None, x)
    refused("places", sp.cache_append, cache, k, k, put(sp, np.zeros((b, 2), np.int32)))
    refused("places", sp.cache_append, cache, k, k, put(sp, np.zeros((b, t), F32)))
    refused("heads alone", sp.cache_append, cache, k, k, places, rotation, x.narrow(0, 0, 2))
    refused("Int32 .rows", sp.cache_append, sp.PagedCache(pool, pool, places), k, k, places)
    refused("last axis", sp.cache_append,
            sp.PagedCache(pool.transpose(2, 3), pool.transpose(2, 3), table),
            put(sp, np.zeros((b, hk, t, page), F32)), put(sp, np.zeros((b, hk, t, page), F32)),
            places)
    lengths = put(sp, np.ones(b, np.int32))
    refused("row for every", sp.cache_attention, x, sp.PagedCache(pool, pool))
    refused("multiple of key", sp.cache_attention, x.narrow(1, 0, 3), cache)
    refused("lengths must be", sp.cache_attention, x, cache, put(sp, np.ones(b + 1, np.int32)))
    refused("without a prefix", sp.cache_attention, x, cache, lengths, None, lengths)
    refused("one dtype", sp.cache_attention, x, cache, lengths, cache, places.reshape([b]))
    refused("multiple of prefixes", sp.cache_attention, x, cache, lengths,
            sp.PagedCache(pool, pool, table.narrow(0, 0, 3)))
    refused("finite", sp.cache_attention, x, cache, lengths, scale=float("nan"))
    large = put(sp, np.zeros((1, 1, 1, 257), F32))
    refused("256", sp.cache_attention, large, sp.PagedCache(large, large))
    logits, scores = put(sp, np.zeros((2, 3, 10), F32)), put(sp, np.zeros((2, 3), F32))
    flags = put(sp, np.zeros((2, 3), np.int32))
    refused("scores", sp.beam_select, logits, scores.transpose(0, 1), 2)
    refused("one dtype", sp.beam_select, logits, put(sp, np.zeros((2, 3), F64)), 2)
    refused("picks", sp.beam_select, logits, scores, 0)
    refused("picks", sp.beam_select, logits, scores, 31)
    refused("picks", sp.beam_select, logits, scores, 65)
    refused("end token", sp.beam_select, logits, scores, 2, 10)
    refused("end token", sp.beam_select, logits, scores, 2, None, flags)
    refused("ended", sp.beam_select, logits, scores, 2, 1, scores)
    refused("64 beams", sp.beam_select, put(sp, np.zeros((1, 65, 4), F32)),
            put(sp, np.zeros((1, 65), F32)), 2)
    refused("equally many", sp.reorder, [scores, logits.narrow(0, 0, 1)], places)
    refused("rows", sp.reorder, [sp.sum(scores)], places)


def test_caches_are_written_at_places_of_their_own(sp):
    """Expanded caches, and one tensor for keys and values, are read but not written."""
    b, hk, d, page = 2, 2, 16, 4
    pool = [put(sp, random((6, hk, page, d), F32, 5 + i)) for i in range(2)]
    one = [x.narrow(1, 0, 1).expand([6, hk, page, d]) for x in pool]
    table = put(sp, np.arange(6, dtype=np.int32).reshape(2, 3))
    x = put(sp, np.ones((b, hk, 1, d), F32))
    places = put(sp, np.zeros((b, 1), np.int32))
    for key, value in ((one[0], pool[1]), (pool[0], one[1]), (pool[0], pool[0]),
                       (pool[0].narrow(0, 0, 1).expand([6, hk, page, d]), pool[1]),
                       (pool[0].narrow(2, 0, 1).expand([6, hk, page, d]), pool[1])):
        with pytest.raises(ValueError, match="places of their own"):
            sp.cache_append(sp.PagedCache(key, value, table), x, x, places)
    got = get(sp, sp.cache_attention(x, sp.PagedCache(*one, table)))
    shared = [np.broadcast_to(get(sp, x.narrow(1, 0, 1)), (6, hk, page, d)) for x in pool]
    held = oracle.Pool(np.zeros((b, hk, 12, d), F32), np.zeros((b, hk, 12, d), F32), [12] * b, page)
    held.table, (held.key, held.value) = get(sp, table), shared
    want, bound = oracle.attention(np.ones((b, hk, 1, d), F32), held)
    assert_within(got, want, bound)
    sp.cache_append(sp.PagedCache(*pool, table), x, x, places)
    assert (get(sp, pool[0])[[0, 3], :, 0] == 1).all() and (get(sp, pool[1])[[0, 3], :, 0] == 1).all()
