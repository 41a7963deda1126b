"""The operators over several sequences under arrays that hold anything: a workspace that stays good, memory around every buffer
that stays as it was, refusals."""
import ctypes

import numpy as np
import pytest

from adaforge_amd import _native as N
from adaforge_amd import hip
from tests import paged_ref as R
from tests.test_gpu_serving import F16, Q4, f32, make_attention, rng_of, run_attention, run_select, same

pytestmark = pytest.mark.gpu
up = hip.Buffer.from_numpy


FALLING = [  # (KV heads, starts, lengths): rows named by several sequences whose keys make different numbers of chunks
    (8, [0, 4, 0, 4, 0], [6000, 0, 2500, 0]),
    (8, [0, 6, 0, 5, 3], [6000, 0, 2500, 3000]),
    (4, [40, 0] * 35 + [40], [0, 3000, 0, 6000] * 17 + [0, 3000]),
]


@pytest.mark.parametrize("q4", [F16, Q4])
@pytest.mark.parametrize("kv,starts,lengths", FALLING)
@pytest.mark.parametrize("width", [64, 128])
def test_a_workspace_after_starts_that_do_not_rise(q4, width, kv, starts, lengths):
    """The rows of such a call may hold anything; its workspace serves the next calls, attention and choice alike."""
    n, qh = len(lengths), 16 * kv
    _, bad, kp, vp, q = make_attention(("fell", int(q4), width, n), q4, width, 64, qh, kv, [1] * n, [6000] * 2 + [64] * (n - 2), tokens=100)
    _, b, kp2, vp2, q2 = make_attention(("next", int(q4), width, n), q4, width, 64, qh, kv, [1] * n, [max(1, 6000 >> (i % 12)) for i in range(n)])
    want = R.attention(b, kp2.values(), vp2.values(), q2, kv, 1 / np.sqrt(width))
    x = f32(rng_of("fell", n), 100, 20000)
    y, result = R.select(x)
    ws = R.workspace(65536 + 524288 * (width + 4))
    for hint in ((1, 6000), (40, 6000)):
        dev, qb, o = R.Device(bad, kp, vp), up(q), up(np.full(q.shape, -7, np.float32))
        dev.keep[0].upload(np.array(starts, np.uint32))
        dev.keep[1].upload(np.array(lengths, np.uint32))
        R.attend(dev, qb, o, qh, 1 / np.sqrt(width), longest=hint, ws=ws)
        for _ in range(2):
            z, ids = run_select(x, ws=ws)
            same(z, y)
            assert np.array_equal(ids, result), hint
            got, _ = run_attention(b, kp2, vp2, q2, kv, ws=ws)
            R.check_attention(got, want, width, 2.0)
