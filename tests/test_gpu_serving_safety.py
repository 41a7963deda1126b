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


def guarded(a):
    """A device buffer with 4,096 bytes in front of and behind the array's, and a function that says whether they are as they were."""
    whole = np.full(a.nbytes + 8192, 0xA5, np.uint8)
    whole[4096:4096 + a.nbytes] = np.ascontiguousarray(a).view(np.uint8).reshape(-1)
    buf = up(whole)

    def read():
        now = buf.numpy()
        assert (now[:4096] == 0xA5).all() and (now[4096 + a.nbytes:] == 0xA5).all()
        return now[4096:4096 + a.nbytes].view(a.dtype).reshape(a.shape)

    return buf, buf.ptr + 4096, read


@pytest.mark.parametrize("q4", [F16, Q4])
@pytest.mark.parametrize("starts,lengths", [([0, 7, 0xFFFFFFFF, 2], [0xFFFFFFFF, 1 << 31, 5]), ([0, 3, 6, 9], [9, 0xFFFFFFFF, 40]),
                                            ([0, 3, 6, 9], [2, 48, 1 << 24]), ([3, 3, 9, 0xFFFFFFFF], [9, 20, 1 << 30])])
def test_wild_arrays_beside_good_pages(q4, starts, lengths):
    """Starts and lengths beyond everything while half of the table names pages: rows are written, none outside the pools and the
    rows, and the rows of a pool that no position names stay as they were."""
    rng = rng_of("beside", int(q4), len(lengths))
    b = R.Batch(rng, [3, 3, 3], [48, 48, 48], 16, tokens=9)
    b.table[:, 1] = [0xFFFFFFF0, b.pages, 0x80000000]
    b.starts[:] = starts
    b.lengths = lengths
    kp, vp = (R.Pool(rng, q4, b.pages, 16, 1, 64) for _ in range(2))
    dev = R.Device(b, kp, vp)
    keep, reads = [], []
    for x in (kp.bytes, vp.bytes, np.full((9, 64), -7, np.float32), np.full((9, 64), -7, np.float32), np.full((9, 1, 64), 9, np.uint16),
              np.full((9, 1, 64), 9, np.uint16)):
        buf, ptr, read = guarded(x)
        keep.append((buf, ptr))
        reads.append(read)
    (_, dev.pages.k), (_, dev.pages.v), (_, qo), (_, out), (_, ko), (_, vo) = keep
    q, k, v = (up(f32(rng, 9, 64)) for _ in range(3))
    a = N.KvAppendArgs(q.ptr, 64, k.ptr, 64, v.ptr, 64, None, None, 1e-6, 1e-6, 1e-6, 0, None, 1, qo, 64, dev.pages, dev.batch)
    N.check(N.lib().af_kv_append(ctypes.byref(a), None))
    N.check(N.lib().af_kv_read(ctypes.byref(dev.pages), ctypes.byref(dev.batch), ko, vo, None))
    t = N.PagedAttentionArgs(qo, 64, out, 64, N.AttentionConfigDesc(1, 1, 64, 0, 0.125), 0, dev.pages, dev.batch, 3, 48, None)
    ws = R.workspace(65536 + 524288 * 68)
    t.workspace = ws.h
    N.check(N.lib().af_paged_attention(ctypes.byref(t), None))
    hip.synchronize()
    after = [r() for r in reads]
    # which pool rows may differ: those that a row's position names (of any sequence whose rows hold it)
    may = np.zeros((b.pages, 16), bool)
    for s in range(3):
        first, stop = min(starts[s], 9), min(starts[s + 1], 9)
        for i in range(first, stop):
            at = b.place(s, min(lengths[s], 1 << 30) - (starts[s + 1] - i))
            if at:
                may[at] = True
    wrote = 0
    for old, new in zip((kp, vp), after[:2]):
        now = R.Pool(rng, q4, b.pages, 16, 1, 64)
        now.bytes[:] = new
        for x, y in zip(old.planes(), now.planes()):
            if x is not None:
                differ = (x.view(np.uint16 if x.dtype == np.float16 else x.dtype) != y.view(np.uint16 if x.dtype == np.float16 else x.dtype)).any((1, 3))
                assert not (differ & ~may).any()
                wrote += int(differ.sum())
    assert (wrote > 0) == may.any()


def test_a_workspace_smaller_than_the_split_needs_is_refused():
    """One sequence of 20,000 positions is split whatever the widths; its sums do not fit the smallest workspace, nor one byte too few."""
    for q4 in (F16, Q4):
        for width in (64, 512):
            _, b, kp, vp, q = make_attention(("split", int(q4)), q4, width, 16, 4, 2, [1], [20000])
            dev, qb, o = R.Device(b, kp, vp), up(q), up(np.full(q.shape, -7, np.float32))
            a = R.attend_args(dev, qb, o, 4, 0.1, longest=(1, 20000))
            size = N.sz()
            N.check(N.lib().af_paged_attention_workspace(ctypes.byref(a), ctypes.byref(size)))
            assert size.value > 65536
            for n in (16, size.value - 1):
                ws = R.workspace(n)
                a.workspace = ws.h
                assert N.lib().af_paged_attention(ctypes.byref(a), None) == N.AF_ERR_INVALID
                assert "workspace" in N.lib().af_last_error().decode()
            ws = R.workspace(size.value)
            a.workspace = ws.h
            N.check(N.lib().af_paged_attention(ctypes.byref(a), None))
            hip.synchronize()
            assert (o.numpy() != -7).all()
