"""The operators over several sequences on the GPU, against plain 64-bit forms: appending to a paged cache, reading it
back, attention over it, the choice of a token, and a step that uses them together."""
import ctypes
import zlib

import numpy as np
import pytest

from adaforge_amd import _native as N
from adaforge_amd import hip
from tests import paged_ref as R

pytestmark = pytest.mark.gpu
F16, Q4 = False, True
up = hip.Buffer.from_numpy


def rng_of(*key):
    return np.random.default_rng([zlib.crc32(k.encode()) if isinstance(k, str) else k for k in key])


def f32(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


def f32_close(got, want):
    """One rounding of a 64-bit result (2^-24 of it); the 64-bit arithmetic before adds 1e-12 of the row's size."""
    want = np.asarray(want, np.float64)
    tol = 2.0 ** -24 * np.abs(want) * (1 + 1e-6) + 1e-12 * np.abs(want).max(initial=0.0) + 2.0 ** -150
    assert (np.abs(got.astype(np.float64) - want) <= tol).all(), np.abs(got - want).max()


# ---- append and read -----------------------------------------------------------------------------

def run_append(batch, kp, vp, q, k, v, q_norm, k_norm, v_norm, rope, eps=(1e-6, 2e-6, 3e-6), pad=0, in_place=False,
               stream=None):
    tokens, qh, w = (batch.tokens, 0, k.shape[2]) if q is None else q.shape
    dev = R.Device(batch, kp, vp)

    def rows(x):  # rows `pad` floats apart, the gaps holding what must not be used
        if x is None:
            return None, 0
        a = np.full((x.shape[0], x.shape[1] * w + pad), 1e9, np.float32)
        a[:, :x.shape[1] * w] = x.reshape(x.shape[0], -1)
        return up(a), a.shape[1]

    (qb, qs), (kb, ks), (vb, vs) = rows(q), rows(k), rows(v)
    ob = None if q is None else qb if in_place else up(np.full((tokens, qs), -7, np.float32))
    norms = [up(n) if n is not None else None for n in (q_norm, k_norm)]
    p = lambda b: b.ptr if b is not None else None  # noqa: E731
    a = N.KvAppendArgs(p(qb), qs, p(kb), ks, p(vb), vs, p(norms[0]), p(norms[1]), *eps, 1 if v_norm else 0,
                       rope.h if rope else None, qh, p(ob), qs, dev.pages, dev.batch)
    N.check(N.lib().af_kv_append(ctypes.byref(a), stream))
    hip.synchronize()
    out = None if q is None else ob.numpy()[:, :qh * w].reshape(tokens, qh, w)
    return dev, out


def expected_append(batch, q, k, v, q_norm, k_norm, v_norm, turn, eps=(1e-6, 2e-6, 3e-6)):
    """{row: (q, k, v)} in 64 bits before any rounding."""
    out = {}
    for row, s, pos in batch.rows():
        r = []
        for x, w, e in ((q, q_norm, eps[0]), (k, k_norm, eps[1])):
            y = None
            if x is not None:
                y = x[row].astype(np.float64)
                y = R.rms(y, w, e) if w is not None else y
                y = R.rotate(y, pos, *turn) if turn else y
            r.append(y)
        y = v[row].astype(np.float64)
        out[row] = (*r, R.rms(y, None, eps[2]) if v_norm else y)
    return out


def check_pool(dev_buf, before, batch, rows, which):
    """The pool holds the rows' values where they belong and is otherwise unchanged."""
    got, want = R.Pool(np.random.default_rng(0), before.q4, before.pages, before.page, before.kv_heads, before.width), before
    got.bytes[:] = dev_buf.numpy()
    if before.q4:
        for row, s, pos in batch.rows():
            at = batch.place(s, pos)
            if at:
                want.put(*at, rows[row][which].astype(np.float32))
        # the f32 value is rounded from 64 bits alike but for ties of 1e-12: no code or scale differs
        assert (got.bytes == want.bytes).all(), np.argwhere(got.bytes != want.bytes)[:5]
        return
    g, w = got.values().copy(), want.values().copy()
    for row, s, pos in batch.rows():
        at = batch.place(s, pos)
        if not at:
            continue
        r = rows[row][which]
        with np.errstate(over="ignore"):
            # fp16's half step (2^-11, or 2^-25 below its normal numbers), after f32's
            tol = 2.0 ** -11 * np.abs(r) * (1 + 2.0 ** -11) + 2.0 ** -25
        assert (np.abs(g[at[0], :, at[1]].astype(np.float64) - r) <= tol).all()
        w[at[0], :, at[1]] = g[at[0], :, at[1]]
    assert np.array_equal(g.view(np.uint16), w.view(np.uint16))


APPENDS = [  # q4, width, page, q_heads, kv_heads, new, lengths
    (F16, 256, 16, 16, 8, [1], [4097]),
    (Q4, 256, 32, 16, 8, [1, 1, 1], [1, 32, 33]),
    (F16, 64, 16, 3, 1, [5, 0, 17, 1], [5, 9, 40, 16]),
    (Q4, 64, 64, 4, 4, [33, 1], [95, 70000]),
    (F16, 128, 128, 6, 2, [129, 2], [131, 257]),
    (Q4, 128, 16, 8, 2, [7, 31, 1, 1], [7, 31, 16, 17]),
    (F16, 512, 256, 16, 1, [3, 20], [131000, 20]),
    (Q4, 512, 16, 2, 1, [19], [65555]),
]


@pytest.mark.parametrize("q4,width,page,qh,kv,new,lengths", APPENDS)
@pytest.mark.parametrize("v_norm", [False, True])
def test_append(q4, width, page, qh, kv, new, lengths, v_norm):
    rng = rng_of(width, page, qh, int(v_norm))
    b = R.Batch(rng, new, lengths, page)
    kp, vp = (R.Pool(rng, q4, b.pages, page, kv, width) for _ in range(2))
    q, k, v = f32(rng, b.tokens, qh, width), f32(rng, b.tokens, kv, width), f32(rng, b.tokens, kv, width)
    qn, kn = 1 + 0.1 * f32(rng, width), 1 + 0.1 * f32(rng, width)
    turn = (1e6, np.linspace(1, 8, width // 2).astype(np.float32))
    dev, out = run_append(b, kp, vp, q, k, v, qn, kn, v_norm, R.rope(width, *turn), pad=8 * v_norm)
    want = expected_append(b, q, k, v, qn, kn, v_norm, turn)
    for row, r in want.items():
        f32_close(out[row], r[0])
    check_pool(dev.k, kp, b, want, 1)
    check_pool(dev.v, vp, b, want, 2)


@pytest.mark.parametrize("q4", [F16, Q4])
def test_append_without_norms_queries_or_rotation(q4):
    rng = rng_of("plain", int(q4))
    b = R.Batch(rng, [4, 3], [40, 3], 16)
    kp, vp = (R.Pool(rng, q4, b.pages, 16, 2, 64) for _ in range(2))
    k, v = f32(rng, b.tokens, 2, 64), f32(rng, b.tokens, 2, 64)
    dev, _ = run_append(b, kp, vp, None, k, v, None, None, False, None)
    want = expected_append(b, None, k, v, None, None, False, None)
    check_pool(dev.k, kp, b, want, 1)
    check_pool(dev.v, vp, b, want, 2)


def test_append_in_place_of_the_queries():
    rng = rng_of("in place")
    b = R.Batch(rng, [9], [9], 16)
    kp, vp = (R.Pool(rng, F16, b.pages, 16, 1, 128) for _ in range(2))
    q, k, v = f32(rng, 9, 5, 128), f32(rng, 9, 1, 128), f32(rng, 9, 1, 128)
    qn = 1 + 0.1 * f32(rng, 128)
    turn = (1e4, np.ones(64, np.float32))
    _, out = run_append(b, kp, vp, q, k, v, qn, None, False, R.rope(128, *turn), pad=4, in_place=True)
    for row, r in expected_append(b, q, k, v, qn, None, False, turn).items():
        f32_close(out[row], r[0])


@pytest.mark.parametrize("q4", [F16, Q4])
def test_append_leaves_out_positions_without_a_page_and_rows_behind_the_last_sequence(q4):
    rng = rng_of("holes", int(q4))
    # sequence 0 has 6 rows but a length of 4 (two rows before position 0); 1 runs past its table; 2 has a bad entry
    b = R.Batch(rng, [6, 5, 4], [4, 50, 20], 16, table_stride=3, tokens=19)
    b.table[2, 1] = b.pages  # one past the last page
    kp, vp = (R.Pool(rng, q4, b.pages, 16, 2, 64) for _ in range(2))
    q, k, v = (f32(rng, 19, h, 64) for h in (2, 2, 2))
    turn = (1e4, np.ones(32, np.float32))
    dev, out = run_append(b, kp, vp, q, k, v, None, None, False, R.rope(64, *turn))
    want = expected_append(b, q, k, v, None, None, False, turn)
    check_pool(dev.k, kp, b, want, 1)
    check_pool(dev.v, vp, b, want, 2)
    assert (out[15:] == -7).all()
    for row, r in want.items():
        f32_close(out[row], r[0])
    got = [hip.Buffer.from_numpy(np.full((19, 2, 64), 0x1234, np.uint16)) for _ in range(2)]
    N.check(N.lib().af_kv_read(ctypes.byref(dev.pages), ctypes.byref(dev.batch), got[0].ptr, got[1].ptr, None))
    hip.synchronize()
    for g, pool in zip(got, (kp, vp)):
        g = g.numpy()
        pool.bytes[:] = (dev.k if pool is kp else dev.v).numpy()
        vals = pool.values()
        for row, s, pos in b.rows():
            at = b.place(s, pos)
            w = vals[at[0], :, at[1]].view(np.uint16) if at else np.zeros((2, 64), np.uint16)
            assert np.array_equal(g[row], w), (row, s, pos)
        assert (g[15:] == 0x1234).all()


def test_wild_arrays_write_nothing_outside():
    """starts that fall, lengths beyond everything, pages that are none: every access stays in its buffers (an index that
    did not would differ in the pools or the guard rows)."""
    rng = rng_of("wild")
    b = R.Batch(rng, [3, 3, 3], [9, 9, 9], 16, tokens=9)
    b.starts = np.array([0, 7, 0xFFFFFFFF, 2], np.uint32)
    b.lengths = [0xFFFFFFFF, 1 << 31, 5]
    b.table[:] = 0xFFFFFFF0
    kp, vp = (R.Pool(rng, F16, b.pages, 16, 1, 64) for _ in range(2))
    before = kp.bytes.copy(), vp.bytes.copy()
    q, k, v = (f32(rng, 9, 1, 64) for _ in range(3))
    dev, out = run_append(b, kp, vp, q, k, v, None, None, False, None)
    assert np.array_equal(dev.k.numpy(), before[0]) and np.array_equal(dev.v.numpy(), before[1])
    o = up(np.full((9, 64), 5, np.float32))
    R.attend(dev, up(q), o, 1, 1.0)
    got = o.numpy()
    assert (got[:9][got[:9] != 5] == 0).all()


def test_four_bit_blocks_at_their_limits():
    """Zeros, subnormal scales, both signs of the largest magnitude, values past fp16, infinities and NaN."""
    rng = rng_of("limits")
    x = np.zeros((8, 1, 64), np.float32)
    x[1, 0, :32] = np.linspace(-1, 1, 32)
    x[1, 0, 32:] = 2.0 ** -24 * np.arange(32)
    x[2, 0, 3], x[2, 0, 9] = 5.0, -5.0          # both signs: the positive one makes the scale
    x[3, 0, 3] = 5.2e5                          # scale just within fp16
    x[3, 0, 40] = 6e5                           # and beyond: NaNs
    x[4, 0, 0] = np.inf
    x[5, 0, 33] = np.nan
    x[6, 0] = rng.standard_normal(64) * 1e-30   # scale 0: zeros
    x[7, 0] = rng.standard_normal(64) * 2.0 ** -20
    b = R.Batch(rng, [8], [8], 16)
    kp, vp = (R.Pool(rng, Q4, b.pages, 16, 1, 64) for _ in range(2))
    dev, _ = run_append(b, kp, vp, None, x, x[::-1].copy(), None, None, False, None)
    for row, s, pos in b.rows():
        kp.put(*b.place(s, pos), x[row])
        vp.put(*b.place(s, pos), x[7 - row])
    for buf, pool in ((dev.k, kp), (dev.v, vp)):
        got = R.Pool(rng, Q4, b.pages, 16, 1, 64)
        got.bytes[:] = buf.numpy()
        for g, w in zip(got.planes(), pool.planes()):
            nan = np.isnan(w) if w.dtype == np.float16 else np.zeros(w.shape, bool)
            assert np.array_equal(g[~nan], w[~nan])
            if nan.any():
                assert np.isnan(g[nan]).all()
        g, w = got.values(), pool.values()
        assert np.array_equal(np.isnan(g), np.isnan(w)) and np.array_equal(g[~np.isnan(w)], w[~np.isnan(w)])


# ---- attention -----------------------------------------------------------------------------------

def make_attention(key, q4, width, page, qh, kv, new, lengths, spread=2.0, fill="random", **kw):
    rng = rng_of(*key)
    b = R.Batch(rng, new, lengths, page, **kw)
    kp, vp = (R.Pool(rng, q4, b.pages, page, kv, width, fill) for _ in range(2))
    return rng, b, kp, vp, (spread * f32(rng, b.tokens, qh, width))


def run_attention(b, kp, vp, q, kv, window=0, sinks=0, longest=None, stream=None, ws=None):
    w, qh = q.shape[2], q.shape[1]
    dev, qb = R.Device(b, kp, vp), up(q)
    o = up(np.full(q.shape, -7, np.float32))
    longest = longest or (max(b.new), max(b.lengths))
    R.attend(dev, qb, o, qh, 1 / np.sqrt(w), window, sinks, longest, ws=ws, stream=stream)
    return o.numpy(), dev


ATTENTIONS = [  # q4, width, page, q_heads, kv_heads, new, lengths, window, sinks
    (F16, 256, 16, 16, 8, [1], [512], 0, 0),
    (F16, 256, 16, 2, 2, [1, 1, 1, 1, 1, 1], [1, 2, 31, 32, 33, 65], 0, 0),
    (Q4, 256, 32, 4, 2, [1, 1, 1, 1], [1, 100, 1000, 2500], 0, 0),
    (F16, 256, 64, 16, 8, [1, 1], [3000, 17], 1024, 4),
    (Q4, 256, 16, 3, 1, [1, 1, 1], [600, 101, 99], 100, 37),
    (F16, 64, 16, 8, 1, [1, 1, 1], [15, 16, 777], 0, 0),
    (Q4, 64, 128, 6, 2, [1, 5, 1], [15, 300, 1500], 0, 0),
    (F16, 128, 32, 12, 4, [1, 2, 9], [1000, 2, 40], 33, 1),
    (Q4, 128, 256, 5, 1, [1, 3], [999, 3], 0, 0),
    (F16, 512, 64, 16, 1, [1, 1], [1100, 64], 0, 0),
    (Q4, 512, 16, 4, 1, [1, 4], [900, 70], 512, 4),
    (Q4, 512, 64, 32, 2, [1, 1], [333, 64], 0, 0),
    (F16, 256, 64, 16, 8, [70], [70], 0, 0),
    (F16, 256, 16, 4, 2, [33, 1, 64, 0, 129], [33, 500, 200, 7, 400], 0, 0),
    (Q4, 256, 32, 6, 2, [100, 31], [350, 31], 0, 0),
    (F16, 64, 16, 8, 2, [150, 17], [400, 17], 64, 5),
    (Q4, 64, 64, 3, 3, [200], [333], 0, 0),
    (F16, 128, 128, 7, 1, [61, 90], [61, 290], 0, 0),
    (Q4, 128, 16, 8, 4, [65, 1], [129, 1200], 100, 0),
    (F16, 512, 32, 16, 1, [40], [200], 0, 0),
    (Q4, 512, 64, 8, 2, [50, 3], [50, 700], 128, 4),
]


@pytest.mark.parametrize("q4,width,page,qh,kv,new,lengths,window,sinks", ATTENTIONS)
def test_attention(q4, width, page, qh, kv, new, lengths, window, sinks):
    _, b, kp, vp, q = make_attention((width, page, qh, len(new), window), q4, width, page, qh, kv, new, lengths)
    got, _ = run_attention(b, kp, vp, q, kv, window, sinks)
    want = R.attention(b, kp.values(), vp.values(), q, kv, 1 / np.sqrt(width), window, sinks)
    R.check_attention(got, want, width, 2.0)


@pytest.mark.parametrize("q4", [F16, Q4])
@pytest.mark.parametrize("new", [[1, 1, 1], [40, 1, 33]])
def test_attention_hints_do_not_change_what_is_computed(q4, new):
    """Hints that are too small or too large, and rows behind the last sequence left as they were."""
    _, b, kp, vp, q = make_attention(("hints", int(q4), len(new), new[0]), q4, 128, 16, 4, 2, new, [700, 1300, 90], tokens=sum(new) + 5)
    want = R.attention(b, kp.values(), vp.values(), q, 2, 1 / np.sqrt(128))
    for longest in [(1, 1), (0, 0), (40, 1300), (1 << 16, 1 << 24), (0xFFFFFFFF, 0xFFFFFFFF), (3, 100)]:
        got, _ = run_attention(b, kp, vp, q, 2, longest=longest)
        R.check_attention(got, want, 128, 2.0)
        assert (got[sum(new):] == -7).all()


@pytest.mark.parametrize("q4,width", [(F16, 64), (Q4, 64), (F16, 256), (Q4, 256), (F16, 512), (Q4, 512)])
@pytest.mark.parametrize("new", [[1], [30], [90]])
def test_attention_over_many_chunks(q4, width, new):
    """Contexts whose keys are split, for single tokens, several row tiles and shared tiles: 1 row of 90 or more at the end
    of 3,000 positions, under a window of 1,500 with 40 first tokens too."""
    _, b, kp, vp, q = make_attention(("chunks", int(q4), width, new[0]), q4, width, 64, 2, 1, new, [3000])
    kv = kp.values(), vp.values()
    for window, sinks in ((0, 0), (1500, 40)):
        got, _ = run_attention(b, kp, vp, q, 1, window, sinks)
        R.check_attention(got, R.attention(b, *kv, q, 1, 1 / np.sqrt(width), window, sinks), width, 2.0)


@pytest.mark.parametrize("q4", [F16, Q4])
@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("hint", [1, 20000])
def test_long_chunks_and_many_of_them(q4, new, hint):
    """One chunk of every key (the page numbers are read again and again), and as many as there may be (128)."""
    _, b, kp, vp, q = make_attention(("long", int(q4), new), q4, 64, 16, 2, 1, [new], [20000])
    got, _ = run_attention(b, kp, vp, q, 1, longest=(new, hint))
    R.check_attention(got, R.attention(b, kp.values(), vp.values(), q, 1, 0.125), 64, 2.0)


@pytest.mark.parametrize("q4,width", [(F16, 64), (Q4, 128), (Q4, 256), (F16, 512)])
@pytest.mark.parametrize("new,lengths", [([1, 1], [2500, 30]), ([1, 0, 1, 1, 1], [200, 900, 0, 3000, 1400]),
                                         ([6, 25, 1, 0, 9], [1000, 2600, 1, 50, 9]),
                                         ([50, 40, 1, 0, 64, 33], [1500, 3000, 2, 40, 64, 900]), ([1] * 64, [1 + 37 * i for i in range(64)])])
def test_sequences_of_very_different_lengths(q4, width, new, lengths):
    """Chunks dealt out by the lengths there are: long beside short and empty ones, one and several row tiles, one more row
    behind the last sequence; with a window too."""
    _, b, kp, vp, q = make_attention(("ragged", int(q4), width, len(new), new[0]), q4, width, 16, 2, 1, new, lengths, tokens=sum(new) + 1)
    kv = kp.values(), vp.values()
    for window, sinks in ((0, 0), (700, 40)):
        want = R.attention(b, *kv, q, 1, 1 / np.sqrt(width), window, sinks)
        for longest in ((max(new), max(lengths)), (1, 300), (max(new), 300), (max(new), 450), (max(new), 1 << 24)):
            got, _ = run_attention(b, kp, vp, q, 1, window, sinks, longest)
            R.check_attention(got, want, width, 2.0)
            assert (got[sum(new):] == -7).all()


@pytest.mark.parametrize("q4,width", [(F16, 256), (F16, 128), (Q4, 256), (Q4, 512), (F16, 64)])
@pytest.mark.parametrize("new", [[24, 17, 1, 20, 24, 9, 3, 23], [16, 9, 1, 10, 0, 2, 12, 16], [29, 32, 0, 31, 8, 25, 30, 2]])
def test_a_few_row_tiles_over_many_keys(q4, width, new):
    """Row tiles of 16 and of 64 rows, whichever the launch takes for these types and widths."""
    lengths = [1100, 40, 700, 1099, 24, 513, 3, 800]
    lengths = [max(n, m) for n, m in zip(lengths, new)]
    _, b, kp, vp, q = make_attention(("tiles", int(q4), width, new[0]), q4, width, 32, 16, 8, new, lengths)
    got, _ = run_attention(b, kp, vp, q, 8)
    R.check_attention(got, R.attention(b, kp.values(), vp.values(), q, 8, 1 / np.sqrt(width)), width, 2.0)


@pytest.mark.parametrize("q4", [F16, Q4])
@pytest.mark.parametrize("sequences,longest", [(70, 3), (70, 60), (5000, 1)])
def test_many_sequences(q4, sequences, longest):
    """More sequences than one round of loads finds (64), some of them without rows."""
    rng = rng_of("sequences", sequences, longest, int(q4))
    new = [1] * sequences if longest == 1 else [int(rng.integers(0, 4)) for _ in range(sequences)]
    if longest > 3:
        new[3] = new[66] = longest
    new[10] = 0
    lengths = [n + int(rng.integers(0, 40)) for n in new]
    _, b, kp, vp, q = make_attention(("sequences", sequences), q4, 64, 16, 4, 2, new, lengths)
    want = R.attention(b, kp.values(), vp.values(), q, 2, 0.125)
    got, _ = run_attention(b, kp, vp, q, 2)
    R.check_attention(got, want, 64, 2.0)
    k, v = f32(rng, b.tokens, 2, 64), f32(rng, b.tokens, 2, 64)
    dev, _ = run_append(b, kp, vp, None, k, v, None, None, False, None)
    rows = expected_append(b, None, k, v, None, None, False, None)
    check_pool(dev.k, kp, b, rows, 1)
    check_pool(dev.v, vp, b, rows, 2)


def test_append_of_a_long_batch():
    """Enough rows that a wave takes four of them."""
    rng = rng_of("long batch")
    for q4, width, qh, kv in ((F16, 128, 13, 2), (Q4, 64, 14, 1)):
        b = R.Batch(rng, [1500, 600], [1500, 900], 64)
        kp, vp = (R.Pool(rng, q4, b.pages, 64, kv, width) for _ in range(2))
        q, k, v = (f32(rng, b.tokens, h, width) for h in (qh, kv, kv))
        qn, kn = 1 + 0.1 * f32(rng, width), 1 + 0.1 * f32(rng, width)
        turn = (1e4, np.ones(width // 2, np.float32))
        dev, out = run_append(b, kp, vp, q, k, v, qn, kn, True, R.rope(width, *turn))
        want = expected_append(b, q, k, v, qn, kn, True, turn)
        for row, r in want.items():
            f32_close(out[row], r[0])
        if not q4:
            check_pool(dev.k, kp, b, want, 1)
            check_pool(dev.v, vp, b, want, 2)
        else:  # (Pool.put packs a whole pool: the rows at once instead)
            got = [R.Pool(rng, q4, b.pages, 64, kv, width) for _ in range(2)]
            for g, buf, which in zip(got, (dev.k, dev.v), (1, 2)):
                g.bytes[:] = buf.numpy()
                w, d = g.planes()
                for row, s, pos in b.rows():
                    n, scale = R.quantise(want[row][which].astype(np.float32))
                    pg, sl = b.place(s, pos)
                    assert np.array_equal(((w[pg, :, sl, :, None] >> R.SHIFT) & 15).reshape(kv, width), n)
                    assert np.array_equal(d[pg, :, sl], scale)


def test_sequences_that_share_pages():
    """A common beginning held once: both sequences' tables name its pages."""
    for q4, new in ((F16, [1, 1]), (Q4, [40, 33])):
        _, b, kp, vp, q = make_attention(("prefix", int(q4)), q4, 128, 16, 4, 2, new, [300, 250])
        b.table[1, :12] = b.table[0, :12]
        got, _ = run_attention(b, kp, vp, q, 2)
        R.check_attention(got, R.attention(b, kp.values(), vp.values(), q, 2, 1 / np.sqrt(128)), 128, 2.0)


@pytest.mark.parametrize("q4", [F16, Q4])
@pytest.mark.parametrize("new", [[6, 3, 2, 1], [70, 80, 40, 66]])
def test_attention_of_missing_keys(q4, new):
    """Rows before position 0 see nothing (zeros), positions past the table or without a page are not seen."""
    lengths = [new[0] - 2, 200, 90, 60]
    _, b, kp, vp, q = make_attention(("missing", int(q4), new[0]), q4, 64, 16, 2, 1, new, lengths, table_stride=10)
    b.table[2, 1] = 0xFFFFFFFF
    b.table[3, :] = b.pages  # no page at all
    got, _ = run_attention(b, kp, vp, q, 1)
    want = R.attention(b, kp.values(), vp.values(), q, 1, 0.125)
    assert (got[:2] == 0).all() and (got[int(b.starts[3]):int(b.starts[4])] == 0).all()
    R.check_attention(got, want, 64, 2.0)


@pytest.mark.parametrize("q4", [F16, Q4])
@pytest.mark.parametrize("new,window", [([1, 1], 0), ([1, 1], 20), ([50, 33], 0), ([50, 33], 20)])
def test_unwritten_pages_are_never_seen(q4, new, window):
    """Every position that no query sees holds NaNs: those past a sequence's length, before its window, and other
    sequences' pages."""
    lengths = [90, 133]
    rng, b, kp, vp, q = make_attention(("unseen", int(q4), new[0], window), q4, 64, 32, 4, 2, new, lengths, fill="nan")
    for s, n in enumerate(lengths):
        lowest = max(0, n - new[s] + 1 - window) if window else 0
        for j in list(range(lowest, n)) + list(range(min(3, lowest))):
            for pool in (kp, vp):
                pool.put(*b.place(s, j), f32(rng, 2, 64))
    got, _ = run_attention(b, kp, vp, q, 2, window, 3)
    want = R.attention(b, kp.values(), vp.values(), q, 2, 0.125, window, 3)
    R.check_attention(got, want, 64, 2.0)


@pytest.mark.parametrize("new,before", [([1, 1], 0), ([45, 18], 0), ([1, 1], 1500), ([45, 18], 1500)])
@pytest.mark.parametrize("where,value", [("v", np.inf), ("k", np.inf), ("k", -np.inf), ("v", np.nan), ("k", np.nan), ("q4 k", np.nan)])
def test_an_infinity_reaches_only_the_positions_that_see_it(new, before, where, value):
    """An overflowed value (an fp16 infinity, or a 4-bit block of NaNs): queries before it are as without it, those that
    see it are as in plain arithmetic (an infinite value in its channel; a key scored -infinity has no weight, one scored
    +infinity makes NaNs)."""
    lengths = [before + 60, before + 200]
    q4 = where.startswith("q4")
    rng, b, kp, vp, q = make_attention(("inf", new[0], where[-1], before), q4, 64, 16, 2, 1, new, lengths)
    pool = vp if where == "v" else kp
    at = b.place(0, before + (50 if new[0] > 1 else 20))
    if q4:
        codes, scales = pool.planes()
        scales[at[0], 0, at[1], 1] = np.nan
        pool._join(codes, scales)
    else:
        pool.planes()[0][at[0], 0, at[1], 7] = value
    got, _ = run_attention(b, kp, vp, q, 1)
    want = R.attention(b, kp.values(), vp.values(), q, 1, 0.125)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(want), np.isnan(got)) and np.array_equal(want == np.inf, got == np.inf)
    assert fine.any()
    w = np.where(fine, want, 0.0)
    g = np.where(fine, got.astype(np.float64), 0.0)
    assert np.linalg.norm(g - w) <= 2 * R.attention_bound(64, 2.0) * np.linalg.norm(w)


@pytest.mark.parametrize("q4,width", [(F16, 128), (Q4, 128), (F16, 256), (Q4, 256), (F16, 512), (Q4, 512)])
@pytest.mark.parametrize("new", [[3, 1], [40, 9]])
def test_not_a_number_among_the_keys_of_every_width(q4, width, new):
    """One key that is no number, seen by some rows of a tile and not by others: those are as without it."""
    rng, b, kp, vp, q = make_attention(("nan", int(q4), width, new[0]), q4, width, 16, 4, 2, new, [700, 90])
    clean = R.attention(b, kp.values(), vp.values(), q, 2, 1 / np.sqrt(width))
    at = b.place(0, 700 - new[0] // 2 - 1)
    if q4:
        codes, scales = kp.planes()
        scales[at[0], 1, at[1], 1] = np.nan
        kp._join(codes, scales)
    else:
        kp.planes()[0][at[0], 1, at[1], 7] = np.nan
    got, _ = run_attention(b, kp, vp, q, 2)
    seen = new[0] - new[0] // 2 - 1  # the first row whose position is the key's
    assert np.isnan(got[seen:new[0], 2:]).all()
    want = clean.copy()
    want[seen:new[0], 2:] = 0
    got[seen:new[0], 2:] = 0
    R.check_attention(got, want, width, 2.0)


@pytest.mark.parametrize("q4", [F16, Q4])
@pytest.mark.parametrize("n", [1, 34])
def test_large_and_small_queries(q4, n):
    """Queries of 1e-30, of 1e4 (one key takes everything) and of zeros (the mean of the values)."""
    rng, b, kp, vp, q = make_attention(("sizes", int(q4), n), q4, 128, 16, 2, 1, [n] * 3, [150, 151, 152])
    q[:n] *= 1e-30
    q[n:2 * n] = 0
    q[2 * n:] *= 5e3
    got, _ = run_attention(b, kp, vp, q, 1)
    want = R.attention(b, kp.values(), vp.values(), q, 1, 1 / np.sqrt(128))
    R.check_attention(got[:2 * n], want[:2 * n], 128, 1.0)
    # scores of up to 5e4: an ulp of them is 2^-8.4, so weights are right to about 1 % and the largest wins
    assert np.abs(got[2 * n:] - want[2 * n:]).max() <= 0.1 * np.abs(want).max()


@pytest.mark.parametrize("q4", [F16, Q4])
@pytest.mark.parametrize("new", [[1, 1], [40, 3]])
def test_strided_rows(q4, new):
    _, b, kp, vp, q = make_attention(("strides", int(q4), new[0]), q4, 64, 16, 4, 2, new, [100, 70])
    dev, t = R.Device(b, kp, vp), b.tokens
    wide = np.full((t, 4 * 64 + 12), np.nan, np.float32)
    wide[:, :256] = q.reshape(t, -1)
    o = up(np.full((t, 4 * 64 + 8), -7, np.float32))
    R.attend(dev, up(wide), o, 4, 0.125, longest=(max(new), 100), strides=(268, 264))
    got = o.numpy()
    assert (got[:, 256:] == -7).all()
    R.check_attention(got[:, :256].reshape(t, 4, 64), R.attention(b, kp.values(), vp.values(), q, 2, 0.125), 64, 2.0)


def test_a_long_cache_past_four_gigabytes():
    """Pages whose byte offsets pass 32 bits: the last pages of a pool of 4.5 GiB."""
    width, page, kv = 256, 256, 8
    per = N.lib().af_kv_page_bytes(N.AF_KV_F16, page, kv, width)
    pages = (9 << 29) // per + 1
    rng = rng_of("long")
    b = R.Batch(rng, [1, 1], [700, 300], page)
    small = [R.Pool(rng, F16, b.pages, page, kv, width) for _ in range(2)]
    big = [hip.Buffer(pages * per, np.uint8) for _ in range(2)]
    first = pages - b.pages
    for pool, buf in zip(small, big):
        N.check(hip.rt().hipMemcpy(buf.ptr + first * per, np.ascontiguousarray(pool.bytes).ctypes.data, pool.bytes.size, hip.H2D))
    q = 2 * f32(rng, 2, 16, width)
    want = R.attention(b, small[0].values(), small[1].values(), q, kv, 1 / 16)
    dev = R.Device(b, *small)
    moved = up(np.where(b.table < b.pages, b.table + np.uint32(first), np.uint32(R.NO_PAGE)))
    dev.pages.k, dev.pages.v, dev.pages.pages, dev.batch.table = big[0].ptr, big[1].ptr, pages, moved.ptr
    o = up(np.zeros(q.shape, np.float32))
    R.attend(dev, up(q), o, 16, 1 / 16, longest=(1, 700))
    R.check_attention(o.numpy(), want, width, 2.0)
    # and the appended rows land there
    k, v = f32(rng, 2, kv, width), f32(rng, 2, kv, width)
    a = N.KvAppendArgs(None, 0, up(k).ptr, kv * width, None, kv * width, None, None, 1e-6, 1e-6, 1e-6, 0, None, 0, None, 0,
                       dev.pages, dev.batch)
    kb, vb = up(k), up(v)
    a.k, a.v = kb.ptr, vb.ptr
    N.check(N.lib().af_kv_append(ctypes.byref(a), None))
    got = [hip.Buffer((2, kv, width), np.float16) for _ in range(2)]
    N.check(N.lib().af_kv_read(ctypes.byref(dev.pages), ctypes.byref(dev.batch), got[0].ptr, got[1].ptr, None))
    hip.synchronize()
    assert np.array_equal(got[0].numpy(), k.astype(np.float16)) and np.array_equal(got[1].numpy(), v.astype(np.float16))


# ---- the choice of a token -------------------------------------------------------------------------

def run_select(x, penalties=None, history=None, bias=None, mask=None, out=True, in_place=False, pad=0, ws=None, stream=None):
    rows, vocab = x.shape
    wide = np.full((rows, vocab + pad), 7e7, np.float32)
    wide[:, :vocab] = x
    keep = [up(wide)]
    ptr = lambda a: keep.append(up(a)) or keep[-1].ptr  # noqa: E731
    ob = None if not out else keep[0] if in_place else up(np.full((rows, vocab + pad), -3, np.float32))
    result = up(np.zeros((rows, 2), np.uint32))
    a = N.LogitsArgs(keep[0].ptr, vocab + pad, ob.ptr if ob else None, vocab + pad, rows, vocab)
    if penalties is not None:
        a.penalties = ptr(np.asarray(penalties, np.float32))
    if history is not None:
        n = max(1, max(len(h) for h in history))
        h = np.zeros((rows, n), np.uint32)
        for r, ids in enumerate(history):
            h[r, :len(ids)] = ids
        a.history, a.history_stride = ptr(h), n
        a.history_len = ptr(np.array([len(h) for h in history], np.uint32))
    if bias is not None:
        n = max(1, max(len(p) for p in bias))
        ids, val = np.zeros((rows, n), np.uint32), np.zeros((rows, n), np.float32)
        for r, p in enumerate(bias):
            for i, (t, v) in enumerate(p):
                ids[r, i], val[r, i] = t, v
        a.bias_ids, a.bias_values, a.bias_stride = ptr(ids), ptr(val), n
        a.bias_len = ptr(np.array([len(p) for p in bias], np.uint32))
    if mask is not None:
        words = (vocab + 31) // 32
        bits = np.zeros((rows, words * 32), bool)
        bits[:, :vocab] = mask
        a.mask = ptr(np.packbits(bits, axis=1, bitorder="little").view(np.uint32))
        a.mask_stride = words
    a.result = result.ptr
    size = N.sz()
    N.check(N.lib().af_logits_select_workspace(ctypes.byref(a), ctypes.byref(size)))
    ws = ws or R.workspace(size.value)
    a.workspace = ws.h
    N.check(N.lib().af_logits_select(ctypes.byref(a), stream))
    hip.synchronize()
    y = ob.numpy() if ob else None
    if ob and not in_place:
        assert (y[:, vocab:] == -3).all()
    return (y[:, :vocab] if ob else None), result.numpy()


def same(got, want):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    f = ~np.isnan(want)
    assert np.array_equal(got[f], want[f]), np.argwhere(got != want)[:5]


def select_inputs(rng, rows, vocab, n_hist, n_bias, allowed):
    x = 3 * f32(rng, rows, vocab)
    hist = [(rng.random(rng.integers(0, n_hist + 1)) ** 4 * vocab).astype(np.uint32) for _ in range(rows)]
    bias = [[(int(rng.integers(0, vocab)), float(np.float32(4 * rng.standard_normal()))) for _ in range(rng.integers(0, n_bias + 1))]
            for _ in range(rows)]
    pen = np.stack([rng.uniform(0.8, 1.5, rows), rng.uniform(-1, 1, rows), rng.uniform(0, 1, rows)], 1).astype(np.float32)
    return x, pen, hist, bias, rng.random((rows, vocab)) < allowed


@pytest.mark.parametrize("rows,vocab,n_hist,n_bias,allowed", [(1, 1, 3, 2, 1.0), (3, 31, 10, 5, 0.5), (2, 33, 100, 0, 0.1),
                                                              (5, 1001, 400, 50, 0.01), (4, 4096, 20, 300, 0.5),
                                                              (2, 32768, 3000, 30, 0.3), (1, 262144, 70, 10, 0.9),
                                                              (17, 50257, 500, 300, 0.001)])
@pytest.mark.parametrize("pad", [0, 1, 4])
def test_select(rows, vocab, n_hist, n_bias, allowed, pad):
    rng = rng_of("select", rows, vocab, pad)
    x, pen, hist, bias, mask = select_inputs(rng, rows, vocab, n_hist, n_bias, allowed)
    want, result = R.select(x, pen, hist, bias, mask)
    for kw in (dict(), dict(in_place=True), dict(out=False)):
        got, ids = run_select(x, pen, hist, bias, mask, pad=pad, **kw)
        assert np.array_equal(ids, result), kw
        if got is not None:
            same(got, want)


def test_select_parts_alone():
    rng = rng_of("alone")
    x, pen, hist, bias, mask = select_inputs(rng, 6, 777, 200, 20, 0.4)
    for kw in (dict(), dict(penalties=pen), dict(history=hist), dict(penalties=pen, history=hist), dict(bias=bias), dict(mask=mask)):
        want, result = R.select(x, **kw)
        got, ids = run_select(x, **kw)
        same(got, want)
        assert np.array_equal(ids, result), kw


def test_select_ties_empty_rows_and_values_that_are_no_numbers():
    x = np.zeros((9, 300), np.float32)
    x[0, [41, 7, 250]] = 2.0                       # a tie: the lowest id
    x[1] = -0.0
    x[1, 100] = 0.0                                # zeros of both signs are equal
    x[2] = -np.inf
    x[3] = np.nan
    x[4, 5] = np.nan
    x[4, 6] = 1.0
    x[5, [9, 12]] = np.inf
    x[6] = -np.finfo(np.float32).max               # the type's lowest value is a value
    x[7, 33], x[7, 34] = np.nan, np.inf            # in masked places
    x[8] = 5.0
    mask = np.ones((9, 300), bool)
    mask[7, [33, 34]] = False
    mask[8] = False                                # nothing allowed
    want, result = R.select(x, mask=mask)
    got, ids = run_select(x, mask=mask)
    same(got, want)
    assert np.array_equal(ids, result)
    assert result[:, 0].tolist() == [7, 0, R.NO_PAGE, R.NO_PAGE, 6, 9, 0, 0, R.NO_PAGE] and result[:, 1].tolist() == [0, 0, 0, 1, 1, 1, 0, 0, 0]


def test_select_ids_twice_and_outside_the_vocabulary():
    rng = rng_of("twice")
    x = f32(rng, 2, 100)
    hist = [[3] * 60000 + [99, 100, 101, 0xFFFFFFFF], []]
    bias = [[(5, 1.0), (6, 2.0), (5, -3.0), (100, 9.0), (0xFFFFFFFF, 9.0), (5, 0.25)], [(0, -np.inf)] * 3]
    pen = [[1.25, 0.5, 0.001], [2.0, 1.0, 1.0]]
    want, result = R.select(x, pen, hist, bias)
    got, ids = run_select(x, pen, hist, bias)
    same(got, want)
    assert np.array_equal(ids, result)


@pytest.mark.parametrize("rows,vocab", [(64, 65536), (600, 5000), (1100, 130)])
def test_select_many_rows(rows, vocab):
    """Enough slices for the narrow blocks, more rows than tickets a line apart, rows of one slice."""
    rng = rng_of("rows", rows)
    x, pen, hist, bias, mask = select_inputs(rng, rows, vocab, 40, 5, 0.5)
    want, result = R.select(x, pen, hist, bias, mask)
    for _ in range(2):
        got, ids = run_select(x, pen, hist, bias, mask)
        same(got, want)
        assert np.array_equal(ids, result)


def test_select_longest_lists():
    rng = rng_of("longest")
    x = f32(rng, 1, 5000)
    hist = [rng.integers(0, 5000, 65535).astype(np.uint32)]
    bias = [[(int(t), float(i)) for i, t in enumerate(rng.integers(0, 5000, 65535))]]
    want, result = R.select(x, [[1.1, 0.1, 0.01]], hist, bias)
    got, ids = run_select(x, [[1.1, 0.1, 0.01]], hist, bias)
    same(got, want)
    assert np.array_equal(ids, result)


# ---- together: streams, graphs, workspaces ---------------------------------------------------------

def test_a_workspace_serves_calls_of_both_kinds_in_turn():
    rng, b, kp, vp, q = make_attention(("shared",), F16, 128, 16, 4, 2, [1, 1, 1], [900, 2000, 10])
    want = R.attention(b, kp.values(), vp.values(), q, 2, 1 / np.sqrt(128))
    x = f32(rng, 8, 20000)
    y, result = R.select(x)
    ws = R.workspace(64 << 20)
    for _ in range(3):
        got, _ = run_attention(b, kp, vp, q, 2, ws=ws)
        R.check_attention(got, want, 128, 2.0)
        z, ids = run_select(x, ws=ws)
        same(z, y)
        assert np.array_equal(ids, result)


def test_a_small_workspace_is_refused():
    _, b, kp, vp, q = make_attention(("small",), F16, 128, 16, 4, 2, [1], [20000])
    dev, qb, o = R.Device(b, kp, vp), up(q), up(np.zeros(q.shape, np.float32))
    a = R.attend_args(dev, qb, o, 4, 0.1, longest=(1, 20000))
    size = N.sz()
    N.check(N.lib().af_paged_attention_workspace(ctypes.byref(a), ctypes.byref(size)))
    if size.value > 65536:
        ws = R.workspace(16)
        a.workspace = ws.h
        assert N.lib().af_paged_attention(ctypes.byref(a), None) == N.AF_ERR_INVALID
        assert "workspace" in N.lib().af_last_error().decode()


@pytest.mark.parametrize("q4", [F16, Q4])
def test_serving_steps_captured_and_replayed(q4):
    """A decode step of three sequences (append, attend, choose) as a graph that follows the lengths in device memory:
    replayed step by step against the same calls made directly, with other work between."""
    rng = rng_of("graph", int(q4))
    w, qh, kv, page, steps, vocab = 128, 4, 2, 16, 5, 3000
    lengths = [30, 400, 15]
    b = R.Batch(rng, [1, 1, 1], [n + steps for n in lengths], page)
    pools = [R.Pool(rng, q4, b.pages, page, kv, w) for _ in range(2)]
    turn = R.rope(w, 1e4, np.ones(w // 2))
    x = [f32(rng, steps, 3, h, w) for h in (qh, kv, kv)]
    logits = f32(rng, steps, 3, vocab)
    norm = up(1 + 0.1 * f32(rng, w))

    def make():
        dev = R.Device(b, *pools)
        s = dict(dev=dev, q=hip.Buffer((3, qh, w)), k=hip.Buffer((3, kv, w)), v=hip.Buffer((3, kv, w)), o=hip.Buffer((3, qh, w)),
                 logits=hip.Buffer((3, vocab)), out=hip.Buffer((3, vocab)), result=hip.Buffer((3, 2), np.uint32))
        s["append"] = N.KvAppendArgs(s["q"].ptr, qh * w, s["k"].ptr, kv * w, s["v"].ptr, kv * w, norm.ptr, norm.ptr, 1e-6, 1e-6,
                                     1e-6, 1, turn.h, qh, s["q"].ptr, qh * w, dev.pages, dev.batch)
        s["attend"] = R.attend_args(dev, s["q"], s["o"], qh, 1 / np.sqrt(w), 64, 4, (1, 450))
        s["select"] = N.LogitsArgs(s["logits"].ptr, vocab, s["out"].ptr, vocab, 3, vocab, result=s["result"].ptr)
        size, most = N.sz(), 0
        for f, a in (("af_paged_attention_workspace", s["attend"]), ("af_logits_select_workspace", s["select"])):
            N.check(getattr(N.lib(), f)(ctypes.byref(a), ctypes.byref(size)))
            most = max(most, size.value)
        s["ws"] = R.workspace(most)
        s["attend"].workspace = s["select"].workspace = s["ws"].h
        return s

    def enqueue(s, stream):
        N.check(N.lib().af_kv_append(ctypes.byref(s["append"]), stream))
        N.check(N.lib().af_paged_attention(ctypes.byref(s["attend"]), stream))
        N.check(N.lib().af_logits_select(ctypes.byref(s["select"]), stream))

    graph_side, plain_side, stream = make(), make(), hip.Stream()
    graph = hip.Graph(stream, lambda: enqueue(graph_side, stream.handle))
    for i in range(steps):
        outs = []
        for s in (graph_side, plain_side):
            s["dev"].keep[1].upload(np.array([n + i + 1 for n in lengths], np.uint32))
            for n, a in zip("qkv", x):
                s[n].upload(a[i])
            s["logits"].upload(logits[i])
            if s is graph_side:
                graph.launch(stream)
                stream.synchronize()
            else:
                enqueue(s, None)
                hip.synchronize()
            outs.append([s[n].numpy() for n in ("o", "out", "result")] + [s["dev"].k.numpy(), s["dev"].v.numpy()])
        for g, p in zip(*outs):
            assert np.array_equal(g.view(np.uint8), p.view(np.uint8)), i
        # and the plain form on what the cache now holds
        held = [R.Pool(rng, q4, b.pages, page, kv, w) for _ in range(2)]
        for h, a in zip(held, outs[1][3:]):
            h.bytes[:] = a
        now = R.Batch.__new__(R.Batch)
        now.__dict__ = {**b.__dict__, "lengths": [n + i + 1 for n in lengths]}
        q = np.stack([R.rotate(R.rms(x[0][i][s].astype(np.float64), norm.numpy(), 1e-6), lengths[s] + i, 1e4, np.ones(w // 2))
                      for s in range(3)]).astype(np.float32)
        R.check_attention(outs[1][0], R.attention(now, held[0].values(), held[1].values(), q, kv, 1 / np.sqrt(w), 64, 4), w, 1.0)
        want, result = R.select(logits[i])
        assert np.array_equal(outs[1][2], result)


@pytest.mark.parametrize("q4,width", [(F16, 256), (Q4, 128)])
def test_captured_attention_follows_the_lengths(q4, width):
    """One graph, replayed over lengths that deal the chunks out quite differently, sequences without rows among them."""
    longest, kv, qh = 4000, 2, 4
    _, b, kp, vp, q = make_attention(("replay", int(q4)), q4, width, 32, qh, kv, [1] * 6, [longest] * 6)
    dev, qb, o, stream = R.Device(b, kp, vp), up(q), up(np.zeros(q.shape, np.float32)), hip.Stream()
    args = R.attend_args(dev, qb, o, qh, 1 / np.sqrt(width), 0, 0, (1, longest))
    size = N.sz()
    N.check(N.lib().af_paged_attention_workspace(ctypes.byref(args), ctypes.byref(size)))
    ws = R.workspace(size.value)
    args.workspace = ws.h
    graph = hip.Graph(stream, lambda: N.check(N.lib().af_paged_attention(ctypes.byref(args), stream.handle)))
    values = kp.values(), vp.values()
    for lengths in ([longest] * 6, [1, 2, 3, 4, 5, 6], [longest, 1, 1, 1, 1, 1], [40, 3999, 0, 700, 0, 64], [longest] * 6, [0] * 6):
        dev.keep[1].upload(np.array(lengths, np.uint32))
        o.upload(np.full(q.shape, -7, np.float32))
        graph.launch(stream)
        stream.synchronize()
        got = o.numpy()
        o.upload(np.full(q.shape, -7, np.float32))
        N.check(N.lib().af_paged_attention(ctypes.byref(args), None))
        hip.synchronize()
        assert np.array_equal(got.view(np.uint32), o.numpy().view(np.uint32)), lengths
        now = R.Batch.__new__(R.Batch)
        now.__dict__ = {**b.__dict__, "lengths": lengths}
        R.check_attention(got, R.attention(now, *values, q, kv, 1 / np.sqrt(width), 0, 0), width, 2.0)


def test_attention_of_arrays_that_do_not_rise_stays_inside():
    """starts that fall, rows named by several sequences, lengths past the table: the pools stay as they are, rows behind
    the batch too, and a fresh workspace serves the next call."""
    _, b, kp, vp, q = make_attention(("falls",), Q4, 64, 16, 4, 2, [3] * 5, [900, 10, 500, 700, 3], tokens=20)
    want = R.attention(b, kp.values(), vp.values(), q, 2, 0.125)
    for starts, lengths in (([0, 15, 0, 15, 0, 15], [900, 900, 900, 900, 900]), ([15, 12, 9, 6, 3, 0], [1 << 31] * 5),
                            ([0, 0xFFFFFFFF, 2, 0xFFFFFFFF, 4, 5], [900, 0, 0xFFFFFFFF, 7, 900]), ([20] * 6, [900] * 5)):
        dev, qb = R.Device(b, kp, vp), up(q)
        dev.keep[0].upload(np.array(starts, np.uint32))
        dev.keep[1].upload(np.array(lengths, np.uint32))
        o = up(np.full(q.shape, -7, np.float32))
        R.attend(dev, qb, o, 4, 0.125, longest=(3, 900))
        o.numpy()
        assert np.array_equal(dev.k.numpy(), kp.bytes) and np.array_equal(dev.v.numpy(), vp.bytes)
    got, _ = run_attention(b, kp, vp, q, 2)
    R.check_attention(got, want, 64, 2.0)
    assert (got[15:] == -7).all()


def test_two_streams_with_a_workspace_each():
    rng, b, kp, vp, q = make_attention(("streams",), F16, 256, 16, 4, 2, [1, 1], [5000, 3000])
    want = R.attention(b, kp.values(), vp.values(), q, 2, 1 / 16)
    dev, qb = R.Device(b, kp, vp), up(q)
    streams = [hip.Stream() for _ in range(2)]
    outs = [up(np.zeros(q.shape, np.float32)) for _ in streams]
    hip.synchronize()
    kept = []
    for _ in range(4):
        for s, o in zip(streams, outs):
            kept.append(R.attend(dev, qb, o, 4, 1 / 16, longest=(1, 5000), stream=s.handle))
    for s, o in zip(streams, outs):
        s.synchronize()
        R.check_attention(o.numpy(), want, 256, 2.0)
    assert np.array_equal(outs[0].numpy(), outs[1].numpy())  # the order of sums does not depend on the run
