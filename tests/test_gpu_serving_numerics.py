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
# its product and sum (2^-24 each), the division and the factor of a join (2^-23 together): below 2^-21.

LARGE = [2.0 ** 20, 2.0 ** 27, 2.0 ** 29, 2.0 ** 32]


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
    assert (np.abs(got - want) <= 2.0 ** -21 * np.abs(want)).all(), np.abs(got - want).max()


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
            assert (np.abs(got[:new[0]] - want) <= 2.0 ** -21 * np.abs(want)).all(), (at, hint, np.abs(got[:new[0]] - want).max())


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
