"""Paged attention where its numbers are extreme: scores so large that fp32 holds them to no less than whole units, one key that
takes nearly all of the weight, query channels far apart in size, and values that are infinite, against 64 bits."""
import numpy as np
import pytest

from tests import paged_ref as R
from tests.test_gpu_serving import F16, Q4, f32, make_attention, rng_of, run_attention

pytestmark = pytest.mark.gpu
FEW, MANY = [2, 1], [90, 3]  # rows: of the kernel of few rows, and of many


def norm_error(got, want):
    return np.linalg.norm(got.astype(np.float64) - want) / np.linalg.norm(want)


# ---- large scores -------------------------------------------------------------------------------------
#
# Where a key takes everything the answer is its value.  What the arithmetic may add: the weight as two fp16 halves (2^-23 of it),
# its products and their sum (2^-23: the matrix unit cuts bits off before it rounds), the division and the factor of a join (2^-23
# together): below 2^-21.  A value below fp16's normal numbers enters the unit with the exponent of 2^-14, and bits are cut off
# there (a b + c measured: wrong by 2^-23 of it from 2^-14 up, 2^-22 at 2^-16, 2^-18 at 2^-20, 2^-14 at 2^-24).

LARGE = [2.0 ** 20, 2.0 ** 27, 2.0 ** 29, 2.0 ** 32]


def is_value(got, want):
    return (np.abs(got - want) <= 2.0 ** -21 * np.maximum(np.abs(want), 2.0 ** -14)).all()


@pytest.mark.parametrize("large", LARGE)
@pytest.mark.parametrize("q4,width", [(F16, 64), (Q4, 64), (F16, 256), (Q4, 256), (F16, 512), (Q4, 128)])
@pytest.mark.parametrize("new", [FEW, MANY])
def test_one_visible_key_of_any_score(new, q4, width, large):
    """A window of one: every row's output is the value at its own position, with scores of both signs about `large`."""
    rng, b, kp, vp, q = make_attention(("own key", width, int(q4), new[0]), q4, width, 16, 4, 2, new, [300, 90])
    k, v = kp.values().astype(np.float64), vp.values().astype(np.float64)
    want = np.zeros(q.shape)
    for row, s, pos in b.rows():
        pg, slot = b.place(s, pos)
        for h in range(4):
            score = q[row, h].astype(np.float64) @ k[pg, h // 2, slot] / np.sqrt(width) * np.log2(np.e)
            q[row, h] *= large * rng.uniform(0.5, 2) / abs(score)
            want[row, h] = v[pg, h // 2, slot]
    got, _ = run_attention(b, kp, vp, q, 2, window=1)
    assert is_value(got, want), np.abs(got - want).max()


@pytest.mark.parametrize("large", LARGE)
@pytest.mark.parametrize("q4,width", [(F16, 64), (Q4, 64), (F16, 256), (Q4, 512)])
@pytest.mark.parametrize("new", [FEW, MANY])
def test_one_key_far_above_the_others(new, q4, width, large):
    """Scores of 0 but for one key, in the first chunk, in the middle or among the last ones; keys split and not."""
    n = 2500
    for at in (0, 1200, n - new[0]):
        rng, b, kp, vp, q = make_attention(("far above", width, int(q4), new[0], at), q4, width, 64, 2, 1, new, [n, 60])
        keys = np.zeros(kp.values().shape, np.float32)
        pg, slot = b.place(0, at)
        keys[pg, 0, slot] = f32(rng, width)
        kp.set(keys)
        key = kp.values()[pg, 0, slot].astype(np.float64)
        for row, s, _ in b.rows():
            if s == 0:
                for h in range(2):
                    score = q[row, h].astype(np.float64) @ key / np.sqrt(width) * np.log2(np.e)
                    q[row, h] *= large * rng.uniform(0.5, 2) / score
        want = vp.values()[pg, 0, slot].astype(np.float64)
        for hint in ((max(new), n), (max(new), 1)):
            got, _ = run_attention(b, kp, vp, q, 1, longest=hint)
            assert is_value(got[:new[0]], want), (at, hint, np.abs(got[:new[0]] - want).max())


@pytest.mark.parametrize("power", [10, 18, 20, 21, 22, 23, 24, 26, 29])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("new", [FEW, MANY])
def test_differences_of_large_scores(new, sign, power):
    """Scores large + j unit of whole j from -3 to 3, exact in fp32 in every sum: the weights are those of the differences, across
    tiles and chunks, whatever is added to all scores."""
    n = 2500
    rng, b, kp, vp, q = make_attention(("differences", new[0]), F16, 64, 64, 2, 1, new, [n, 60])
    large, unit = sign * 2.0 ** power, max(1.0, 2.0 ** (power - 23))
    keys = np.zeros(kp.values().shape, np.float32)
    keys[..., 0] = 1
    keys[..., 1] = rng.integers(-3, 4, keys.shape[:-1])
    kp.set(keys)
    q[:] = 0
    q[..., 0], q[..., 1] = 8 * large, 8 * unit
    want = R.attention(b, kp.values(), vp.values(), q, 1, 0.125)
    for hint in ((max(new), n), (max(new), 1)):
        got, _ = run_attention(b, kp, vp, q, 1, longest=hint)
        # The exponential's argument is rounded at up to 16 (2^-21), or at up to 32 where two maxima meet (2^-20).  A sum of n
        # weighted values, one by one in 32 bits: a partial sum has grown to sqrt(k / n) of the last and is rounded uniformly within
        # half an ulp, 2^-24 at most, so that n of them add up to 2^-24 / sqrt(3) sqrt(n / 2); three times that.
        bound = 2.0 ** -19 + 3 * 2.0 ** -24 / np.sqrt(3) * np.sqrt(n / 2)
        assert norm_error(got, want) <= bound, (hint, norm_error(got, want), bound)


# ---- one key that takes nearly all of the weight -------------------------------------------------------

def sunk(key, q4, width, new, n, share, rng_new=None):
    """Sequence 0 of n positions whose first key, of value zero, takes about `share` of every row's weight: the output is what the
    others add.  The first key's score is one product, s0 for every row; the others' are about N(0, 1)."""
    rng, b, kp, vp, q = make_attention(key, q4, width, 64, 2, 1, new, [n, 60], spread=1.0)
    keys, values = f32(rng, *kp.values().shape), f32(rng, *vp.values().shape)
    keys[..., 0] = 0
    pg, slot = b.place(0, 0)
    keys[pg, :, slot] = 0
    keys[pg, :, slot, 0] = 8
    values[pg, :, slot] = 0
    kp.set(keys)
    vp.set(values)
    s0 = np.log(n * np.exp(0.5) * share / (1 - share))
    q[..., 0] = s0 * np.sqrt(width) / 8
    return b, kp, vp, q, s0


@pytest.mark.parametrize("share", [0.5, 0.97, 0.996, 0.9995, 0.9999])
@pytest.mark.parametrize("q4,width", [(F16, 64), (Q4, 64), (F16, 256), (Q4, 128), (F16, 512)])
@pytest.mark.parametrize("new", [FEW, MANY])
def test_a_first_key_that_takes_nearly_all_of_the_weight(new, q4, width, share):
    """First tokens that draw the attention and add nothing: what remains of the output keeps its digits.

    Bound: that of 32-bit scores and sums, the first key's score once more for every row (2^-24 s0 and as much for its exponential's
    argument), and for the keys of its tile, whose weights are held to 2^-38 of the largest there (one 78th of the keys,
    their errors uniform): 3 times 2^-38 / sqrt(3) over their mean weight."""
    n = 2500
    b, kp, vp, q, s0 = sunk(("sink", int(q4), width, new[0]), q4, width, new, n, share)
    want = R.attention(b, kp.values(), vp.values(), q, 1, 1 / np.sqrt(width))
    mean = (1 - share) / n / share
    bound = R.attention_bound(width, 1.0) + 2.0 ** -23 * s0 + 3 * 2.0 ** -38 / np.sqrt(3) / mean * np.sqrt(32 / n)
    for hint in ((max(new), n), (max(new), 1)):
        got, _ = run_attention(b, kp, vp, q, 1, longest=hint)
        rows = slice(0, new[0])
        assert norm_error(got[rows], want[rows]) <= bound, (hint, norm_error(got[rows], want[rows]), bound)


@pytest.mark.parametrize("new", [FEW, MANY])
@pytest.mark.parametrize("q4", [F16, Q4])
def test_tiles_of_very_different_scores(new, q4):
    """Keys' scores in steps of 40 from tile to tile, up and down, the high ones of value zero but for one in a few: sums that grow
    and shrink by e^40 again and again, and a row that sees only the low tiles."""
    n, width = 1500, 64
    rng, b, kp, vp, q = make_attention(("steps", new[0], int(q4)), q4, width, 64, 2, 1, new, [n, 60], spread=1.0)
    for order in range(3):
        keys, values = f32(rng, *kp.values().shape), f32(rng, *vp.values().shape)
        level = np.arange(-(-n // 32))
        level = [level % 2, level * 5 % 7, (level == 20) * 6][order]
        for j in range(n):
            pg, slot = b.place(0, j)
            keys[pg, :, slot, 0] = level[j // 32]
            if level[j // 32] and order != 1:
                values[pg, :, slot] = 0
        keys[..., 0] *= 8
        kp.set(keys)
        vp.set(values)
        q[..., 0] = 40 * np.sqrt(width) / 8
        want = R.attention(b, kp.values(), vp.values(), q, 1, 0.125)
        # (where the high tiles' values are zero the rows' outputs are e^-40 and e^-240 of a value: 32-bit scores of up to 240 have
        # errors of 2^-24 240 in the weights, and the scores' differences across tiles are rounded at up to 350)
        bound = R.attention_bound(width, 1.0) + 2 * 2.0 ** -24 * 350
        for hint in ((max(new), n), (max(new), 1)):
            got, _ = run_attention(b, kp, vp, q, 1, longest=hint)
            g, w = got[:new[0]].astype(np.float64), want[:new[0]]
            if order == 2:  # all of the weight is the high tile's, and its values are zeros
                assert np.abs(g).max() <= 2.0 ** -100
                continue
            assert norm_error(g, w) <= bound, (order, hint, norm_error(g, w), bound)


# ---- query channels far apart in size -------------------------------------------------------------------

@pytest.mark.parametrize("times", [1e3, 1e5, 3e6])
@pytest.mark.parametrize("q4,width", [(F16, 64), (Q4, 64), (F16, 256), (Q4, 512)])
@pytest.mark.parametrize("new", [FEW, MANY])
def test_a_query_channel_far_above_the_others(new, q4, width, times):
    """One channel many times the others, where the keys are zero: the scores are the others' and keep their digits.

    Bound: that of 32-bit arithmetic, and for the small channels of a query, held to 2^-40 of its largest (errors uniform), what they
    add to a score: 3 times 2^-40 / sqrt(3) times the largest, over scores of 2."""
    rng, b, kp, vp, q = make_attention(("outlier", int(q4), width, new[0]), q4, width, 16, 2, 1, new, [700, 60])
    keys = f32(rng, *kp.values().shape)
    keys[..., 5] = 0
    kp.set(keys)
    assert (kp.values()[..., 5] == 0).all()
    q[..., 5] = times * 2
    want = R.attention(b, kp.values(), vp.values(), q, 1, 1 / np.sqrt(width))
    got, _ = run_attention(b, kp, vp, q, 1)
    bound = R.attention_bound(width, 2.0) + 3 * 2.0 ** -40 / np.sqrt(3) * times * 2
    assert norm_error(got, want) <= bound, (norm_error(got, want), bound)


# ---- infinite values that later keys outweigh --------------------------------------------------------------

@pytest.mark.parametrize("new", [FEW, MANY])
@pytest.mark.parametrize("at,above", [(3, 40), (3, 140), (3, 500), (600, 700)])
def test_an_infinite_value_without_weight(new, at, above):
    """An infinite value of a key that another outweighs by e^1000: it has no weight in 64 bits either, and the output is finite,
    whether one wave or block takes both keys or not."""
    n, width = 1000, 64
    rng, b, kp, vp, q = make_attention(("outweighed", new[0], at), F16, width, 64, 2, 1, new, [n, 60], spread=1.0)
    keys = f32(rng, *kp.values().shape)
    keys[..., 0] = 0
    pg, slot = b.place(0, above)
    keys[pg, :, slot, 0] = 8
    kp.set(keys)
    pg, slot = b.place(0, at)
    vp.planes()[0][pg, 0, slot, 7] = np.inf
    q[..., 0] = 1000
    want = R.attention(b, kp.values(), vp.values(), q, 1, 0.125)
    assert np.isfinite(want).all()
    for hint in ((max(new), n), (max(new), 1)):
        got, _ = run_attention(b, kp, vp, q, 1, longest=hint)
        assert np.isfinite(got).all(), hint
        assert norm_error(got, want) <= R.attention_bound(width, 1.0) + 2.0 ** -23 * 1000
