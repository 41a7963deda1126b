"""Plain 64-bit forms of the operators over several sequences (paged cache, attention, token choice), and device calls of
the framework's own through ctypes."""
import ctypes

import numpy as np

from adaforge_amd import _native as N
from adaforge_amd import hip

NO_PAGE = 0xFFFFFFFF


# ---- 4-bit blocks ------------------------------------------------------------------------------

SHIFT = np.array([0, 16, 4, 20, 8, 24, 12, 28], np.uint32)


def quantise(x):
    """Codes [..., w] and fp16 scales [..., w / 32] of f32 rows x."""
    b = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        high, low = b.max(-1), b.min(-1)
        d = (np.where(high >= -low, high, low) / np.float32(-8)).astype(np.float16)
        d = np.where(np.isfinite(b).all(-1) & np.isfinite(d), d, np.float16(np.nan)).astype(np.float16)
        ratio = b.astype(np.float64) / d.astype(np.float64)[..., None]
        n = np.where((d == 0)[..., None] | np.isnan(d)[..., None], 8, np.clip(np.rint(ratio) + 8, 0, 15))
    return n.astype(np.uint8).reshape(x.shape), d


def stands_for(n, d):
    v = (n.astype(np.float32) - np.float32(8)).reshape(*n.shape[:-1], -1, 32) * d.astype(np.float32)[..., None]
    with np.errstate(over="ignore"):
        return v.astype(np.float16).reshape(n.shape)


class Pool:
    """A pool of pages on the host: bytes [pages][kv_heads][part], and the values they stand for."""

    def __init__(self, rng, q4, pages, page, kv_heads, width, fill="random"):
        self.q4, self.page, self.kv_heads, self.width, self.pages = q4, page, kv_heads, width, pages
        part = page * width * 9 // 16 if q4 else page * width * 2
        self.bytes = np.zeros((pages, kv_heads, part), np.uint8)
        if fill == "random":
            self.set(rng.standard_normal((pages, kv_heads, page, width)).astype(np.float32))
        else:  # nothing that was ever written: NaNs
            self.bytes[:] = 0x7F
            if not q4:
                self.bytes[..., 1::2] = 0x7E

    def planes(self):
        if not self.q4:
            return self.bytes.view(np.float16).reshape(self.pages, self.kv_heads, self.page, self.width), None
        cut = self.page * self.width // 2
        shape = (self.pages, self.kv_heads, self.page, -1)
        return (np.ascontiguousarray(self.bytes[..., :cut]).view(np.uint32).reshape(shape),
                np.ascontiguousarray(self.bytes[..., cut:]).view(np.float16).reshape(shape))

    def values(self):
        a, d = self.planes()
        if d is None:
            return a
        return stands_for(((a[..., None] >> SHIFT) & 15).astype(np.uint8).reshape(*a.shape[:-1], -1), d)

    def _join(self, a, d):
        flat = (self.pages, self.kv_heads, -1)
        self.bytes[:] = np.concatenate([np.ascontiguousarray(a).view(np.uint8).reshape(flat),
                                        np.ascontiguousarray(d).view(np.uint8).reshape(flat)], 2)

    def set(self, x):
        if not self.q4:
            with np.errstate(over="ignore"):
                self.planes()[0][:] = x.astype(np.float16)
            return
        n, d = quantise(x)
        w = (n.reshape(*n.shape[:-1], -1, 8).astype(np.uint32) << SHIFT).sum(-1, dtype=np.uint32)
        self._join(w, d)

    def put(self, page, slot, x):
        """Rows x [kv_heads][width] (f32) at a slot."""
        if not self.q4:
            with np.errstate(over="ignore"):
                self.planes()[0][page, :, slot] = x.astype(np.float16)
            return
        n, d = quantise(x)
        w, s = self.planes()
        w[page, :, slot] = (n.reshape(*n.shape[:-1], -1, 8).astype(np.uint32) << SHIFT).sum(-1, dtype=np.uint32)
        s[page, :, slot] = d
        self._join(w, s)


class Batch:
    """Sequences of `new` rows each at the end of `lengths` positions, their pages anywhere in the pool."""

    def __init__(self, rng, new, lengths, page, spare=2, table_stride=None, tokens=None):
        need = [max(0, -(-n // page)) for n in lengths]
        self.page, self.new, self.lengths = page, list(new), list(lengths)
        self.pages = sum(need) + spare
        self.table_stride = table_stride or max(1, max(need) + 1)
        self.table = np.full((len(new), self.table_stride), NO_PAGE, np.uint32)
        order = rng.permutation(self.pages)
        at = 0
        for s, n in enumerate(need):
            k = min(n, self.table_stride)
            self.table[s, :k] = order[at:at + k]
            at += n
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        self.tokens = tokens or max(1, int(self.starts[-1]))

    def place(self, s, p):
        """(page, slot) of position p of sequence s, or None."""
        if p < 0 or p // self.page >= self.table_stride or self.table[s, p // self.page] >= self.pages:
            return None
        return int(self.table[s, p // self.page]), p % self.page

    def rows(self):
        """(row, sequence, position) of every row."""
        for s, (n, length) in enumerate(zip(self.new, self.lengths)):
            for i in range(n):
                yield int(self.starts[s]) + i, s, length - n + i


# ---- the operators -----------------------------------------------------------------------------

def rms(x, w, eps):
    r = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
    return r if w is None else r * w.astype(np.float64)


def rotate(x, pos, base, factors):
    half = x.shape[-1] // 2
    a = float(pos) * np.float64(base) ** (-np.arange(half) / half) / factors.astype(np.float64)
    u, v = x[..., :half], x[..., half:]
    return np.concatenate([u * np.cos(a) - v * np.sin(a), u * np.sin(a) + v * np.cos(a)], -1)


def sees(p, j, window, sinks):
    return (j <= p) & ((window == 0) | (p - j < window) | (j < sinks))


def attention(batch, k, v, q, kv_heads, scale, window=0, sinks=0):
    """[tokens][q_heads][w] in 64 bits over page values k, v; rows that no sequence has are NaN."""
    tokens, qh, w = q.shape
    out, G = np.full(q.shape, np.nan), qh // kv_heads
    for s in range(len(batch.new)):
        n, new, first = batch.lengths[s], batch.new[s], int(batch.starts[s])
        if new == 0:
            continue
        at = [(j, *batch.place(s, j)) for j in range(max(0, n)) if batch.place(s, j) is not None]
        key, pg, sl = (np.array(c, int) for c in zip(*at)) if at else (np.zeros(0, int),) * 3
        K, V = k[pg, :, sl].astype(np.float64), v[pg, :, sl].astype(np.float64)
        pos = n - new + np.arange(new)
        seen = sees(pos[:, None], key[None], window, sinks) & (pos[:, None] >= 0)
        for h in range(qh):
            with np.errstate(all="ignore"):
                x = q[first:first + new, h].astype(np.float64) @ K[:, h // G].T * scale
                x = np.where(seen, x, -np.inf)
                top = x.max(1, initial=-np.inf, keepdims=True)
                e = np.where(seen, np.exp(x - np.where(top == -np.inf, 0.0, top)), 0.0)
                # a key without weight adds nothing, whatever its value
                bad = ~np.isfinite(V[:, h // G]).all(1)
                o = e[:, ~bad] @ V[~bad, h // G]
                for j in np.nonzero(bad)[0]:
                    o += np.where(e[:, j:j + 1] != 0, e[:, j:j + 1] * V[j, h // G], 0.0)
                total = e.sum(1, keepdims=True)
                out[first:first + new, h] = np.where(total == 0, 0.0, o / total)
    return out


def select(x, penalties=None, history=None, bias=None, mask=None):
    """Rows after penalties [rows][3], lists of ids, lists of (id, value), and allowed [rows][vocab]; ids and flags."""
    y = x.astype(np.float64)
    for r in range(x.shape[0]):
        if penalties is not None and history is not None:
            rep, pres, freq = (np.float64(np.float32(v)) for v in penalties[r])
            for t, c in zip(*np.unique([t for t in history[r] if t < x.shape[1]], return_counts=True)):
                t = int(t)
                with np.errstate(all="ignore"):
                    y[r, t] = (y[r, t] / rep if y[r, t] > 0 else y[r, t] * rep) - (freq * c + pres)
        for t, b in dict(bias[r] if bias is not None else []).items():
            if t < x.shape[1]:
                y[r, t] += np.float64(np.float32(b))
    with np.errstate(over="ignore"):
        y = y.astype(np.float32)
    if mask is not None:
        y = np.where(mask, y, np.float32(-np.inf))
    result = np.empty((x.shape[0], 2), np.uint32)
    for r in range(x.shape[0]):
        c = np.where(np.isnan(y[r]), -np.inf, y[r])
        result[r] = NO_PAGE if c.max() == -np.inf else int(np.argmax(c)), bool((np.isnan(y[r]) | (y[r] == np.inf)).any())
    return y, result


# ---- device calls --------------------------------------------------------------------------------

class Handle:
    def __init__(self, create, free):
        self.h, self._free = N.P(), free
        N.check(create(ctypes.byref(self.h)))

    def __del__(self):
        self._free(self.h)


def workspace(nbytes):
    return Handle(lambda h: N.lib().af_workspace_create(nbytes, h), N.lib().af_workspace_free)


def rope(width, base, factors, context=1 << 20):
    f = np.ascontiguousarray(factors, np.float32)
    d = N.RopeDesc(width, base, f.ctypes.data_as(N.f32p), context)
    return Handle(lambda h: N.lib().af_rope_create(ctypes.byref(d), h), N.lib().af_rope_free)


class Device:
    """Buffers of a batch and its pools, and the structs that name them."""

    def __init__(self, batch, k_pool, v_pool):
        up = hip.Buffer.from_numpy
        self.keep = [up(batch.starts), up(np.asarray(batch.lengths, np.int64).astype(np.uint32)), up(batch.table)]
        self.k, self.v = up(k_pool.bytes), up(v_pool.bytes)
        kind = N.AF_KV_Q4 if k_pool.q4 else N.AF_KV_F16
        self.pages = N.KvPages(self.k.ptr, self.v.ptr, kind, k_pool.pages, k_pool.page, k_pool.kv_heads, k_pool.width)
        self.batch = N.KvBatch(*(b.ptr for b in self.keep), batch.table_stride, len(batch.new), batch.tokens)


def attend_args(dev, q, out, q_heads, scale, window=0, sinks=0, longest=(0, 0), strides=None):
    w, kv = dev.pages.width, dev.pages.kv_heads
    sq, so = strides or (q_heads * w, q_heads * w)
    return N.PagedAttentionArgs(q.ptr, sq, out.ptr, so, N.AttentionConfigDesc(q_heads, kv, w, window, scale), sinks,
                                dev.pages, dev.batch, longest[0], longest[1], None)


def attend(dev, q, out, q_heads, scale, window=0, sinks=0, longest=(0, 0), strides=None, ws=None, stream=None):
    a = attend_args(dev, q, out, q_heads, scale, window, sinks, longest, strides)
    size = N.sz()
    N.check(N.lib().af_paged_attention_workspace(ctypes.byref(a), ctypes.byref(size)))
    ws = ws or workspace(size.value)
    a.workspace = ws.h
    N.check(N.lib().af_paged_attention(ctypes.byref(a), stream))
    if stream is None:
        hip.synchronize()
    return ws


def attention_bound(w, s_rms):
    """Relative 2-norm error that 32-bit arithmetic explains.  A score of magnitude s_rms is summed over w products:
    the rounding of a partial sum that has grown to a share x of the terms is uniform within half an ulp,
    2^-25 s_rms sqrt(x) times at most 2, sqrt(w / 2) of them add up to 2^-24 / sqrt(3) sqrt(w / 2) s_rms; two such
    errors enter a weight (score and normalisation).  Operands of 22 bits and the exponential's ulp add 2^-22.
    Three times that."""
    return 3.0 * (2.0 ** -24 * 0.58 * np.sqrt(w / 2) * s_rms * np.sqrt(2) + 2.0 ** -22)


def check_attention(got, want, w, s_rms):
    """Against 64-bit rows `want` (NaN rows: not the call's)."""
    rows = ~np.isnan(want).all((1, 2))
    g, r = got[rows].astype(np.float64), want[rows]
    assert np.isfinite(g).all()
    scale = np.linalg.norm(r) or 1.0
    rel = np.linalg.norm(g - r) / scale
    bound = attention_bound(w, s_rms)
    rms_ = scale / np.sqrt(r.size)
    worst = (np.abs(g - r) / np.maximum(np.abs(r), rms_)).max()
    assert rel <= bound and worst <= 40 * bound, (rel, worst, bound)
