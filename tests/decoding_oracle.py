"""The decoding operators in 64 bits (numpy): caches in pages, attention behind a shared
prefix and beam selection, with bounds on what their kernels may differ by."""
from __future__ import annotations

import numpy as np

from tests.attention_oracle import half_step


# ------------------------------------------------------------------- pages

class Pool:
    """[rows, heads, tokens, extent] keys and values laid into pages.

    page 0: no table, row b is page b.  Pages come in a random order with `spare` pages
    between them that no table names; entries behind a row's length are `behind`, and
    tokens of no row hold `garbage`."""

    def __init__(self, key, value, lengths, page, seed=0, spare=2, behind=-1, garbage=np.nan):
        rng = np.random.default_rng(seed)
        self.rows, self.heads, self.room, self.extent = key.shape
        self.page_tokens = page or max(self.room, 1)
        self.lengths = np.clip(np.asarray(lengths, np.int64), 0, self.room)
        if page == 0:
            self.table, count = None, self.rows
            numbers = np.arange(self.rows)[:, None]
        else:
            entries = -(-self.room // page)
            self.table = np.full((self.rows, entries), behind, np.int32)
            used = np.arange(entries) < -(-self.lengths // page)[:, None]
            count = int(used.sum()) + spare
            self.table[used] = rng.permutation(count)[:used.sum()]
            numbers = self.table
        shape = (count, self.heads, self.page_tokens, self.extent)
        self.key = np.full(shape, garbage, key.dtype)
        self.value = np.full(shape, garbage, key.dtype)
        for b in range(self.rows):
            for t in range(self.lengths[b]):
                at = numbers[b, t // self.page_tokens], slice(None), t % self.page_tokens
                self.key[at], self.value[at] = key[b, :, t], value[b, :, t]
        if page:
            self.room = entries * page

    def tokens(self, row, count):
        """[heads, count, extent] keys and values of the row's first tokens, and which of
        them are there."""
        at = np.arange(min(count, self.room))
        pages = (np.full(at.shape, row) if self.table is None
                 else self.table[row, at // self.page_tokens])
        there = (pages >= 0) & (pages < len(self.key))
        pages, slots = np.where(there, pages, 0), at % self.page_tokens
        return (self.key[pages, :, slots].swapaxes(0, 1),
                self.value[pages, :, slots].swapaxes(0, 1), there)


# --------------------------------------------------------------- attention

def attention(query, cache, lengths=None, prefix=None, prefix_lengths=None, scale=None,
              dtype=np.float32):
    """(output, bound) of queries [batch, heads, queries, extent] over Pools.

    The bound counts roundings (u = half a step).  A score: its products and their sum
    (d u of the products' sizes), the scale in q and log2(e) (3 u).  A weight: its score
    and the row's base, each as far off as a score and u of itself, once more where the
    parts of a row meet; the exponentials (2 x 4 u).  Sums over s keys: a rounding each,
    and one for every part and wave that is joined, which are fewer than 64 + s / 16."""
    b, h, t, d = query.shape
    u = half_step(dtype)
    group = h // cache.heads
    scale = 1 / np.sqrt(d) if scale is None else scale
    rooms = np.full(b, cache.room)
    lengths = rooms if lengths is None else np.clip(np.asarray(lengths, np.int64), 0, cache.room)
    output, bound = np.zeros(query.shape), np.zeros(query.shape)
    for i in range(b):
        key, value, there = cache.tokens(i, lengths[i])
        seen = np.broadcast_to(there, (t, len(there)))
        p = lengths[i] - t + np.arange(t)
        seen = seen & (np.arange(len(there)) <= p[:, None])
        if prefix is not None:
            row = i // (b // prefix.rows)
            count = prefix.room if prefix_lengths is None else int(
                np.clip(prefix_lengths[row], 0, prefix.room))
            first, second, there = prefix.tokens(row, count)
            key, value = np.concatenate([first, key], 1), np.concatenate([second, value], 1)
            seen = np.concatenate([there & (p >= 0)[:, None], seen], 1)
        used = seen.any(0)
        key = np.repeat(key[:, used].astype(np.float64), group, 0)
        value = np.repeat(value[:, used].astype(np.float64), group, 0)
        seen = seen[:, used]
        q = np.where(seen.any(-1)[:, None], query[i].astype(np.float64), 0.0)
        s = seen.shape[1]
        if s == 0:
            continue
        scores = np.where(seen, scale * (q @ key.swapaxes(1, 2)), -np.inf)
        top = scores.max(-1, keepdims=True)
        e = np.exp(scores - np.where(np.isneginf(top), 0.0, top))
        total = e.sum(-1, keepdims=True)
        weights = e / np.where(total == 0, 1.0, total)
        output[i] = weights @ value
        size = np.where(seen, abs(scale) * (np.abs(q) @ np.abs(key).swapaxes(1, 2)), 0.0)
        size = size.max(-1, keepdims=True)
        weight = u * (2 * (d + 4) * size + 8 * size + s + 16)
        bound[i] = (weights @ np.abs(value)) * (2 * weight + u * (2 * s + 96))
    return output, bound


# ------------------------------------------------------------------- beams

def log_sums(logits):
    """log(sum(exp)) of rows, NaN where a NaN or +infinity stands.  Summed in extended
    precision: along an axis that is not the innermost in memory numpy adds term by term,
    which puts 60000 equal terms off by 1.4e-13 in double."""
    x = np.asarray(logits, np.float64)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        top = x.max(-1, keepdims=True)
        total = np.exp(x - top).sum(-1, keepdims=True, dtype=np.longdouble)
        return (top + np.log(total)).astype(np.float64)[..., 0]


def select(logits, scores, picks, ended=None, end_token=-1):
    """(totals, parents, tokens, ended) of [groups, beams, vocabulary] logits."""
    x, score = np.asarray(logits, np.float64), np.asarray(scores, np.float64)
    groups, beams, v = x.shape
    with np.errstate(invalid="ignore"):
        totals = score[..., None] + (x - log_sums(x)[..., None])
    totals[np.isnan(totals)] = -np.inf
    if ended is not None:
        alone = np.full(totals.shape, -np.inf)
        alone[..., end_token] = np.where(np.isnan(score), -np.inf, score)
        totals = np.where((np.asarray(ended) != 0)[..., None], alone, totals)
    made = [np.empty((groups, picks)), *(np.empty((groups, picks), np.int64) for _ in range(3))]
    row, token = (a.ravel() for a in np.indices((beams, v)))
    for g in range(groups):
        total, logit = totals[g].ravel(), np.nan_to_num(x[g].ravel(), nan=-np.inf)
        # totals of -infinity come in the order of rows and tokens alone
        logit = np.where(np.isneginf(total), 0.0, logit)
        order = np.lexsort((token, -logit, row, -total))[:picks]
        made[0][g], made[2][g] = total[order], token[order]
        made[1][g] = g * beams + row[order]
        made[3][g] = token[order] == end_token
        if ended is not None:
            made[3][g] |= np.asarray(ended)[g, row[order]] != 0
    return made


def select_bound(logits, dtype):
    """How far a total may be off before it is rounded: log(sum)'s error.  Terms are exp(x -
    top) with the difference's rounding and that of its product with log2(e) (2 u of the
    range each) and the function's 4 u; sums of 16 in a lane 16 u; a rescaling (the same
    exponential, its differences at most the range in all) for each chunk of 1024 and the
    last to the row's top; the rest is in double.  Rows without a finite logit: 0."""
    x = np.asarray(logits, np.float64)
    finite = x[np.isfinite(x)]
    reach = float(finite.max() - finite.min()) if finite.size else 0.0
    chunks = -(-x.shape[-1] // 512)
    return half_step(dtype) * (8 * reach + 24 + 6 * chunks) + 1e-14


def border(logits, scores, picks, ended=None, end_token=-1):
    """The smallest distance between totals of different rows among a group's best
    picks + 1, which decides whether rounding can change the order."""
    x = np.asarray(logits, np.float64)
    groups, beams, v = x.shape
    more = min(picks + 1, beams * v)
    totals, parents, _, _ = select(logits, scores, more, ended, end_token)
    least = np.inf
    for g in range(groups):
        for i in range(more):
            for j in range(i):
                if parents[g, i] != parents[g, j] and np.isfinite(totals[g, i]):
                    least = min(least, abs(totals[g, i] - totals[g, j]))
    return least
