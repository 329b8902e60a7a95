"""Beam selection and the reordering of states, through the C ABI, against their
definitions in 64 bits."""
import numpy as np
import pytest

from tests import decoding_oracle as oracle
from tests.attention_oracle import half_step

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


def select(hip, logits, scores, picks, ended=None, end_token=-1, gap=0, offset=0):
    groups, beams, v = logits.shape
    dtype = logits.dtype
    whole = np.full(offset + groups * beams * (v + gap), 1e30, dtype)  # would win
    whole[offset:].reshape(groups, beams, v + gap)[..., :v] = logits
    flags = None if ended is None else device(hip, np.asarray(ended, np.int32)).ptr
    shape = hip.beams(groups, beams, v, picks, v + gap, flags, end_token, hip.dtype_tag(dtype))
    need = hip.beam_select_workspace(shape)
    n = groups * picks
    made = [space(hip, dtype.itemsize * n), space(hip, 8 * n), space(hip, 8 * n), space(hip, 4 * n)]
    hip.call("spar_hip_launch_beam_select", *(x.ptr for x in made),
             device(hip, whole).address(offset * dtype.itemsize),
             device(hip, scores.astype(dtype)).ptr, shape, space(hip, need).ptr, need, 0)
    return [x.to_numpy(kind, (groups, picks))
            for x, kind in zip(made, (dtype, np.int64, np.int64, np.int32))]


def check(hip, logits, scores, picks, ended=None, end_token=-1, **more):
    want = oracle.select(logits, scores, picks, ended, end_token)
    off = oracle.select_bound(logits, logits.dtype)
    # rounding must not decide between rows
    assert oracle.border(logits, scores, picks, ended, end_token) > 2 * off
    got = select(hip, logits, scores, picks, ended, end_token, **more)
    for x, y, name in zip(got[1:], want[1:], ("parents", "tokens", "ended")):
        assert np.array_equal(x, y), name
    finite = np.isfinite(want[0])
    assert np.array_equal(got[0][~finite], want[0][~finite])
    bound = half_step(logits.dtype) * np.abs(want[0][finite]) + off
    assert (np.abs(got[0][finite] - want[0][finite]) <= bound).all()


def inputs(groups, beams, v, dtype, seed):
    rng = np.random.default_rng(seed)
    logits = (3 * rng.standard_normal((groups, beams, v))).astype(dtype)
    return logits, (-5 * rng.random((groups, beams))).astype(dtype)


CASES = [  # groups, beams, vocabulary, picks
    (1, 1, 1, 1), (1, 1, 5, 1), (1, 1, 5, 5), (3, 2, 7, 4), (2, 4, 63, 8), (1, 8, 64, 8),
    (5, 3, 1000, 6), (2, 5, 1025, 10), (1, 4, 5003, 4), (2, 1, 30011, 64), (1, 16, 2049, 32),
    (1, 64, 3, 64), (2, 64, 100, 64), (7, 8, 4096, 16), (1, 2, 131075, 3), (40, 8, 1100, 8),
]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("dtype", [F32, F64])
def test_select(hip, case, dtype):
    logits, scores = inputs(*case[:3], dtype, 11)
    check(hip, logits, scores, case[3])


@pytest.mark.parametrize("groups", [1, 600])
def test_many_rows_take_a_wave_each(hip, groups):
    logits, scores = inputs(groups, 8, 515, F32, 12)
    check(hip, logits, scores, 5)


@pytest.mark.parametrize("dtype", [F32, F64])
@pytest.mark.parametrize("gap,offset", [(1, 1), (5, 3)])
def test_rows_with_gaps(hip, dtype, gap, offset):
    logits, scores = inputs(2, 3, 2777, dtype, 13)
    check(hip, logits, scores, 7, gap=gap, offset=offset)


@pytest.mark.parametrize("dtype", [F32, F64])
@pytest.mark.parametrize("order", ["rising", "falling", "equal", "steps", "zeros"])
@pytest.mark.parametrize("picks", [1, 7, 64])
def test_orders_and_equal_logits(hip, dtype, order, picks):
    """Every logit better than all before it, none, and equal ones, of which the lowest
    tokens count, over many chunks of one row; the other row is far behind."""
    v = 20000
    row = {"rising": np.arange(v) / 4096, "falling": -np.arange(v) / 4096, "equal": np.full(v, 2.5),
           "steps": np.arange(v) // 500 % 3 * 0.5,
           "zeros": np.where(np.arange(v) % 3 == 0, -0.0, 0.0)}[order]
    logits = np.stack([row, row - 1])[None].astype(dtype)
    check(hip, logits, np.array([[-1.0, -40.0]]), picks)


@pytest.mark.parametrize("dtype", [F32, F64])
def test_equal_rows_go_by_their_number(hip, dtype):
    """All beams alike: totals of the same bits, the lowest row first."""
    logits = np.broadcast_to(inputs(1, 1, 3000, dtype, 14)[0], (2, 4, 3000)).astype(dtype)
    got = select(hip, logits, np.zeros((2, 4)), 10)
    want = oracle.select(logits, np.zeros((2, 4)), 10)
    for x, y in zip(got[1:3], want[1:3]):
        assert np.array_equal(x, y)


@pytest.mark.parametrize("dtype", [F32, F64])
def test_first_step(hip, dtype):
    """Equal beams of which the first alone counts."""
    logits = np.broadcast_to(inputs(1, 1, 300, dtype, 15)[0], (3, 5, 300)).astype(dtype)
    scores = np.full((3, 5), -np.inf)
    scores[:, 0] = 0
    check(hip, logits, scores, 5)


@pytest.mark.parametrize("dtype", [F32, F64])
@pytest.mark.parametrize("kept", [0, 1, 3, 20])
def test_masked_vocabulary(hip, dtype, kept):
    """Fewer tokens than picks are allowed: the rest are the first rows and tokens."""
    rng = np.random.default_rng(16)
    logits, scores = inputs(2, 3, 2500, dtype, 16)
    allowed = rng.permutation(2500)[:kept]
    masked = np.full(logits.shape, -np.inf, dtype)
    masked[:, 1, allowed] = logits[:, 1, allowed]
    check(hip, masked, scores, 8)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("dtype", [F32, F64])
def test_undefined_rows_lose(hip, dtype, bad):
    """A NaN or +infinity leaves its row no log-softmax: -infinity for all its tokens."""
    logits, scores = inputs(2, 3, 1500, dtype, 17)
    logits[0, 1, 700] = bad
    logits[1, :, 3] = bad
    check(hip, logits, scores, 6)


@pytest.mark.parametrize("score", [np.nan, np.inf, -np.inf])
def test_undefined_scores(hip, score):
    logits, scores = inputs(1, 3, 800, F32, 18)
    scores[0, 1] = score
    check(hip, logits, scores, 4)


@pytest.mark.parametrize("dtype", [F32, F64])
def test_lowest_and_largest_values(hip, dtype):
    """Masks of the type's lowest value, and logits of its largest."""
    logits, scores = inputs(2, 2, 1030, dtype, 19)
    logits[0, :, 5:] = np.finfo(dtype).min
    logits[1, 0, 9] = np.finfo(dtype).max
    want = oracle.select(logits, scores, 7)
    got = select(hip, logits, scores, 7)
    for x, y in zip(got[1:3], want[1:3]):
        assert np.array_equal(x, y)


@pytest.mark.parametrize("dtype", [F32, F64])
def test_ended_beams(hip, dtype):
    logits, scores = inputs(4, 4, 901, dtype, 20)
    ended = np.array([[0, 1, 0, 0], [7, 0, -1, 0], [1, 1, 1, 1], [0, 0, 0, 0]])
    scores[1, 0] = -0.25
    scores[2, 3] = -np.inf
    logits[ended != 0] = np.nan  # rows of ended beams are not used
    check(hip, logits, scores, 6, ended, end_token=450)
    logits, scores = inputs(2, 2, 64, dtype, 21)
    check(hip, logits, scores, 9, None, end_token=3)


# ------------------------------------------------------------------ reorder

@pytest.mark.parametrize("rows,source", [(1, 1), (6, 6), (10, 5), (3, 9)])
def test_reorder(hip, rows, source):
    """States of many widths, types and strides in one call; rows without a parent become
    zeros."""
    rng = np.random.default_rng(22)
    parents = rng.integers(0, source, rows)
    if rows > 5:
        parents[[2, 4]] = -1, source
    states = []
    for i, (width, gap, offset, kind) in enumerate([
            (1, 0, 0, np.int32), (4, 0, 0, F32), (7, 2, 1, np.int64), (1000, 0, 0, F64),
            (5000, 0, 0, F32), (4097, 3, 1, F32), (0, 0, 0, F32), (2, 2, 2, np.int64)] * 5):
        whole = rng.integers(-9, 9, offset + source * (width + gap)).astype(kind)
        target = np.full(offset + rows * (width + gap), 77, kind)
        states.append((width, gap, offset, kind, whole, target, device(hip, whole),
                       device(hip, target)))
    hip.call("spar_hip_launch_reorder", hip.reorders(*(
        (to.address(offset * kind().itemsize), width + gap,
         source_buffer.address(offset * kind().itemsize), width + gap, width, kind().itemsize)
        for width, gap, offset, kind, _, _, source_buffer, to in states)), len(states),
        device(hip, parents.astype(np.int64)).ptr, rows, source, 0)
    for width, gap, offset, kind, whole, target, _, to in states:
        before = whole[offset:].reshape(source, width + gap)
        want = target.copy()
        made = want[offset:].reshape(rows, width + gap)
        for i, p in enumerate(parents):
            made[i, :width] = before[p, :width] if 0 <= p < source else 0
        assert np.array_equal(to.to_numpy(kind, target.shape), want)


@pytest.mark.parametrize("dtype", [F32, F64])
@pytest.mark.parametrize("beams,picks", [(64, 64), (64, 3), (7, 64)])
def test_more_equal_totals_than_are_held_at_once(hip, dtype, beams, picks):
    """All totals of a group are the same: the first tokens of its first beam."""
    logits = np.zeros((2, beams, 20000), dtype)
    scores, parents, tokens, _ = select(hip, logits, np.full((2, beams), -1.5), picks)
    assert (parents == np.array([[0], [beams]])).all()
    assert (tokens == np.arange(picks)).all()
    total = -1.5 - np.log(20000.0)
    bound = half_step(dtype) * abs(total) + oracle.select_bound(logits, dtype)
    assert (np.abs(scores - total) <= bound).all()


@pytest.mark.parametrize("place", [0, 2047, 2048, 4999])
@pytest.mark.parametrize("dtype", [F32, F64])
def test_one_logit_outweighs_all(hip, dtype, place):
    """Its total is its score; others of the row follow far behind."""
    logits, scores = inputs(1, 2, 5000, dtype, 23)
    logits[0, 1, place] = 500
    check(hip, logits, scores, 5)


@pytest.mark.parametrize("dtype", [F32, F64])
@pytest.mark.parametrize("beams,picks", [(16, 32), (16, 64), (3, 17), (64, 16)])
def test_long_parts_of_rows(hip, dtype, beams, picks):
    """Parts of many chunks each, since a group's candidates are bounded."""
    logits, scores = inputs(1, beams, 90001, dtype, 24)
    check(hip, logits, scores, picks)


@pytest.mark.parametrize("dtype", [F32, F64])
@pytest.mark.parametrize("order", ["rising", "falling", "equal", "steps"])
def test_orders_in_long_parts(hip, dtype, order):
    """The bar that a chunk sets for the next ones: each better, each worse, equal ones."""
    v, beams = 60000, 16
    row = {"rising": np.arange(v) / 8192, "falling": -np.arange(v) / 8192,
           "equal": np.full(v, 2.5), "steps": np.arange(v) // 2500 % 4 * 0.5}[order]
    logits = np.broadcast_to(row, (1, beams, v)).astype(dtype)
    scores = -40.0 * np.arange(beams)[None]
    check(hip, logits, scores, 64)


@pytest.mark.parametrize("dtype", [F32, F64])
@pytest.mark.parametrize("vocabulary", [700, 20011])
def test_rows_closer_than_rounding(hip, dtype, vocabulary):
    """Beams with the same logits in other orders: which of them comes first is up to the
    rounding of their sums, but nothing further off than that is chosen or left out, and every
    call chooses alike."""
    beams, picks = 6, 20
    rng = np.random.default_rng(33)
    row = (3 * rng.standard_normal(vocabulary)).astype(dtype)
    logits = np.stack([np.stack([row[rng.permutation(vocabulary)] for _ in range(beams)])
                       for _ in range(3)])
    scores = np.full((3, beams), -2.0)
    totals = scores[..., None] + logits - oracle.log_sums(logits)[..., None]
    off = oracle.select_bound(logits, dtype)
    got = select(hip, logits, scores, picks)
    for again in range(2):
        for x, y in zip(select(hip, logits, scores, picks), got):
            assert np.array_equal(x, y)
    for g in range(3):
        at = got[1][g] - g * beams, got[2][g]
        assert len(set(zip(*at))) == picks
        chosen = totals[g][at]
        assert (np.abs(got[0][g] - chosen) <= off + half_step(dtype) * np.abs(chosen)).all()
        assert (np.diff(got[0][g]) <= 0).all()
        assert (chosen[:-1] >= chosen[1:] - 2 * off).all()
        rest = totals[g].copy()
        rest[at] = -np.inf
        assert rest.max() <= chosen.min() + 2 * off
