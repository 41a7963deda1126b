"""The operators over several sequences, on the CPU: arguments refused before any GPU work, and the index arithmetic
that keeps the kernels in bounds (paged.h, compiled for the host)."""
import ctypes
import os
import random
import subprocess

import pytest

from adaforge_amd import _native as N

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 20  # an aligned address that no call here reads


def refused(rc, word=""):
    msg = N.lib().af_last_error().decode()
    assert rc == N.AF_ERR_INVALID and word in msg, (rc, msg)


def pages(**kw):
    d = dict(k=A, v=2 * A, type=N.AF_KV_F16, pages=8, page=16, kv_heads=2, width=64)
    d.update(kw)
    return N.KvPages(**d)


def batch(**kw):
    d = dict(starts=A, lengths=A, table=A, table_stride=4, sequences=2, tokens=3)
    d.update(kw)
    return N.KvBatch(**d)


def test_page_bytes():
    f = N.lib().af_kv_page_bytes
    assert f(N.AF_KV_F16, 16, 8, 256) == 8 * 16 * 256 * 2
    assert f(N.AF_KV_Q4, 32, 2, 64) == 2 * 32 * (32 + 4)
    for bad in [(2, 16, 8, 256), (0, 8, 8, 256), (0, 512, 8, 256), (0, 24, 8, 256), (0, 16, 0, 256), (0, 16, 1025, 256),
                (0, 16, 8, 96), (0, 16, 8, 0)]:
        assert f(*bad) == 0, bad


BAD_PAGES = [dict(k=None), dict(v=None), dict(k=A + 8), dict(type=2), dict(pages=0), dict(page=24), dict(page=8),
             dict(kv_heads=0), dict(width=96)]
BAD_BATCH = [dict(starts=None), dict(lengths=None), dict(table=None), dict(table_stride=0),
             dict(table_stride=N.AF_MAX_POSITIONS // 16 + 1), dict(sequences=0), dict(sequences=N.AF_MAX_SEQUENCES + 1),
             dict(tokens=0), dict(tokens=N.AF_MAX_BATCH_TOKENS + 1)]


def append_args(p=None, b=None, **kw):
    d = dict(q=A, q_stride=256, k=A, k_stride=128, v=A, v_stride=128, q_norm=A, k_norm=A, q_eps=1e-6, k_eps=1e-6, v_eps=1e-6,
             v_norm=1, rope=None, q_heads=4, q_out=2 * A, q_out_stride=256)
    d.update(kw)
    return N.KvAppendArgs(pages=p or pages(), batch=b or batch(), **d)


@pytest.mark.parametrize("kw", [dict(k=None), dict(v=None), dict(q=None), dict(q_heads=0), dict(q_out=None), dict(q=A + 4),
                                dict(k_stride=126), dict(k_stride=64), dict(q_stride=252), dict(q_out_stride=128),
                                dict(q_out=A, q_out_stride=512), dict(q_heads=1025, q_stride=1 << 20, q_out_stride=1 << 20),
                                dict(q_eps=0.0), dict(k_eps=-1.0), dict(v_eps=float("nan"))], ids=str)
def test_append_refuses(kw):
    refused(N.lib().af_kv_append(ctypes.byref(append_args(**kw)), None))


def test_pages_and_batches_are_checked_by_every_call():
    lib = N.lib()
    for kw in BAD_PAGES:
        refused(lib.af_kv_append(ctypes.byref(append_args(p=pages(**kw))), None))
        refused(lib.af_kv_read(ctypes.byref(pages(**kw)), ctypes.byref(batch()), A, A, None))
        refused(lib.af_paged_attention(ctypes.byref(attention_args(p=pages(**kw))), None))
    for kw in BAD_BATCH:
        refused(lib.af_kv_append(ctypes.byref(append_args(b=batch(**kw))), None))
        refused(lib.af_kv_read(ctypes.byref(pages()), ctypes.byref(batch(**kw)), A, A, None))
        refused(lib.af_paged_attention(ctypes.byref(attention_args(b=batch(**kw))), None))
    refused(lib.af_kv_append(None, None))
    refused(lib.af_kv_read(ctypes.byref(pages()), ctypes.byref(batch()), None, A, None))
    refused(lib.af_kv_read(ctypes.byref(pages()), ctypes.byref(batch()), A, A + 2, None), "aligned")


def attention_args(p=None, b=None, config=(4, 2, 64, 0, 0.125), **kw):
    d = dict(q=A, q_stride=256, out=2 * A, out_stride=256, sinks=0, longest_query=1, longest_context=64, workspace=None)
    d.update(kw)
    return N.PagedAttentionArgs(config=N.AttentionConfigDesc(*config), pages=p or pages(), batch=b or batch(), **d)


@pytest.mark.parametrize("kw", [dict(q=None), dict(out=None), dict(q=A + 4), dict(q_stride=128), dict(out_stride=255),
                                dict(out=A), dict(workspace=None),
                                dict(config=(4, 2, 128, 0, 0.125)), dict(config=(4, 4, 64, 0, 0.125)),
                                dict(config=(3, 2, 64, 0, 0.125)), dict(config=(0, 2, 64, 0, 0.125)),
                                dict(config=(4, 2, 64, 0, 0.0)), dict(config=(4, 2, 64, 0, float("nan"))),
                                dict(config=(2048, 2, 64, 0, 0.1), q_stride=1 << 18, out_stride=1 << 18)], ids=str)
def test_attention_refuses(kw):
    refused(N.lib().af_paged_attention(ctypes.byref(attention_args(**kw)), None))


def test_attention_workspace_asks_for_sizes_alone():
    size = N.sz()
    N.check(N.lib().af_paged_attention_workspace(ctypes.byref(attention_args(q=None, out=None)), ctypes.byref(size)))
    assert size.value > 0
    refused(N.lib().af_paged_attention_workspace(ctypes.byref(attention_args()), None))


def test_one_workspace_fits_every_attention_of_a_width():
    rng, need = random.Random(6), ctypes.c_size_t()
    pick = lambda *c: rng.choice(c)
    for _ in range(20000):
        width, kv = pick(64, 128, 256, 512), pick(1, 2, 3, 8, 16, 100, 1024)
        group = pick(1, 2, 5, 16, 1024 // kv) if kv < 1024 else 1
        qh = kv * group if kv * group <= 1024 else kv
        b = batch(sequences=pick(1, 2, 3, 8, 64, 65, 1000, 4096, rng.randint(1, 4096)), tokens=pick(1, 4, 64, 512, 65536, rng.randint(1, 65536)),
                  table_stride=pick(1, 100, 1 << 16))
        a = attention_args(p=pages(kv_heads=kv, width=width, type=pick(N.AF_KV_F16, N.AF_KV_Q4), page=16), b=b,
                           config=(qh, kv, width, pick(0, 1, 1024), 0.125), sinks=pick(0, 4),
                           longest_query=pick(0, 1, 16, 600, 0xFFFFFFFF), longest_context=pick(0, 1, 500, 8192, 0xFFFFFFFF))
        assert N.lib().af_paged_attention_workspace(ctypes.byref(a), ctypes.byref(need)) == N.AF_OK
        assert need.value <= 65536 + 524288 * (width + 4)


def logits_args(**kw):
    d = dict(logits=A, stride=100, out=None, out_stride=0, rows=2, vocabulary=100, penalties=A, history=A, history_stride=5,
             history_len=A, bias_ids=A, bias_values=A, bias_stride=5, bias_len=A, mask=A, mask_stride=4, result=A,
             workspace=None)
    d.update(kw)
    return N.LogitsArgs(**d)


@pytest.mark.parametrize("kw", [dict(logits=None), dict(result=None), dict(rows=0), dict(rows=N.AF_MAX_LOGIT_ROWS + 1),
                                dict(vocabulary=0), dict(vocabulary=(1 << 24) + 1, stride=1 << 25), dict(stride=99),
                                dict(out=2 * A, out_stride=99), dict(out=A, out_stride=104), dict(history_len=None),
                                dict(history_stride=0), dict(history_stride=65536), dict(bias_values=None),
                                dict(bias_len=None), dict(bias_stride=0), dict(bias_stride=65536), dict(mask_stride=3),
                                dict(workspace=None)], ids=str)
def test_select_refuses(kw):
    refused(N.lib().af_logits_select(ctypes.byref(logits_args(**kw)), None))


def test_rope_refuses():
    f = (ctypes.c_float * 32)(*([1.0] * 32))
    h = N.P()
    for width, base, factors, context in [(0, 1e4, f, 8), (63, 1e4, f, 8), (64, 1.0, f, 8), (64, float("inf"), f, 8),
                                          (64, 1e4, None, 8), (64, 1e4, f, 0),
                                          (64, 1e4, (ctypes.c_float * 32)(*([1.0] * 31 + [0.0])), 8)]:
        refused(N.lib().af_rope_create(ctypes.byref(N.RopeDesc(width, base, factors, context)), ctypes.byref(h)))
    refused(N.lib().af_rope_create(None, ctypes.byref(h)))
    refused(N.lib().af_workspace_create(100, None))


SOURCE = r'''
#include <initializer_list>
#include "paged.h"
using namespace af;
extern "C" {
void span(uint32_t start, uint32_t stop, uint32_t length, uint32_t tokens, uint32_t stride, uint32_t shift, int64_t* o) {
    PagedBatch b{}; b.tokens = tokens; b.table_stride = stride; b.page_shift = shift;
    Span s = span_of(start, stop, length, b);
    o[0] = s.first; o[1] = s.count; o[2] = s.pos0; o[3] = s.end;
}
uint32_t tiles(int32_t plo, int32_t phi, uint32_t end, uint32_t window, uint32_t sinks, uint32_t t, uint32_t* at, uint32_t most) {
    Tiles x = t == 32 ? tiles_of<32>(plo, phi, end, window, sinks) : tiles_of<64>(plo, phi, end, window, sinks);
    for (uint32_t i = 0; i < x.count && i < most; ++i) at[i] = tile_at(x, i);
    return x.count;
}
int see(int32_t p, int32_t j, uint32_t window, uint32_t sinks) { return sees(p, j, window, sinks); }
// chunks a KV head's blocks are dealt, most of a row tile, blocks and bytes there are, bytes that many chunks need
void shares(uint32_t sequences, uint32_t tokens, uint32_t heads, uint32_t group, uint32_t width, uint32_t query, uint32_t context,
            const uint32_t* rows, const uint32_t* keys, uint64_t* o) {
    const AttnPlan p = attn_plan(AttnShape{sequences, tokens, heads, group, width, 0, 0, query, context, 1u << 24});
    uint32_t tiles[64];
    for (uint32_t i = 0; i < sequences; ++i) tiles[i] = (rows[i] * group + p.rows - 1) / p.rows;
    o[0] = o[1] = o[4] = o[5] = 0;
    o[2] = p.shares.chunks;
    o[3] = p.part_bytes;
    if (!p.shares.chunks) return;
    uint32_t total = 0, row_tiles = 0;
    for (uint32_t i = 0; i < sequences; ++i) total += tiles[i] * keys[i], row_tiles += tiles[i];
    o[5] = row_tiles;
    for (uint32_t per : {p.shares.per_fill, p.shares.per_safe}) {
        o[0] = o[1] = 0;
        for (uint32_t i = 0; i < sequences; ++i) {
            const uint32_t chunk = share_chunk(share_of(p.shares, total, per), keys[i]), c = (keys[i] + chunk - 1) / chunk;
            o[0] += tiles[i] * most(1, c);
            o[1] = most((uint32_t)o[1], c);
        }
        if (o[0] <= p.shares.most) break;
    }
    o[4] = o[2] * heads * p.rows * (width + 4) * 4;
}
}
'''


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    (d / "paged.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "adaforge_amd", "csrc"),
                    str(d / "paged.cpp"), "-o", str(d / "paged.so")], check=True)
    return ctypes.CDLL(str(d / "paged.so"))


def test_spans_stay_in_the_batch_whatever_the_arrays_hold(index):
    rng, o = random.Random(3), (ctypes.c_int64 * 4)()
    wild = [0, 1, 2, 7, 100, 65535, 65536, 1 << 24, (1 << 30) - 1, 1 << 30, 1 << 31, 0xFFFFFFFF]
    for _ in range(20000):
        start, stop, length = (rng.choice(wild + [rng.randint(0, 300)]) for _ in range(3))
        tokens, shift = rng.choice([1, 3, 64, 300, 65536]), rng.randint(4, 8)
        stride = rng.choice([1, 4, (1 << 24) >> shift])
        index.span(start, stop, length, tokens, stride, shift, o)
        first, count, pos0, end = o
        assert 0 <= first <= tokens and 0 <= count <= tokens - first
        assert end <= stride << shift and end <= length
        assert -(1 << 30) <= pos0 <= 1 << 30
        if start < stop <= tokens and length < 1 << 30:
            assert (first, count, pos0) == (start, stop - start, length - (stop - start))


def test_tiles_are_those_that_hold_a_seen_key(index):
    rng, at = random.Random(4), (ctypes.c_uint32 * 4096)()
    for _ in range(4000):
        t = rng.choice([32, 64])
        plo = rng.randint(-3, 500)
        phi = plo + rng.randint(0, 70)
        end = rng.choice([0, 1, 5, rng.randint(0, 700)])
        window = rng.choice([0, 0, 1, 2, 31, 32, 33, 100, 1024, 0xFFFFFFFF])
        sinks = rng.choice([0, 0, 1, 4, 32, 33, 70, 1000, 0xFFFFFFFF])
        n = index.tiles(plo, phi, end, window, sinks, t, at, 4096)
        got = list(at[:n])
        assert got == sorted(set(got)) and all(g * t < max(end, 1) for g in got)
        need = {j // t for p in range(max(plo, 0), phi + 1) for j in range(min(p + 1, end)) if index.see(p, j, window, sinks)}
        assert need <= set(got), (plo, phi, end, window, sinks, t)
        assert len(got) <= len(need) + 2 + 70 // t


def test_shared_chunks_fit_their_blocks(index):
    rng, o, dealt = random.Random(5), (ctypes.c_uint64 * 6)(), [0, 0]
    for _ in range(6000):
        n, group, heads = rng.choice([2, 3, 8, 63, 64, rng.randint(2, 64)]), rng.choice([1, 2, 16, 31]), rng.choice([1, 2, 5, 8, 100, 1024])
        rows = [rng.choice([0, 1, 1, 1, 5, rng.randint(0, 60)]) for _ in range(n)]
        top = rng.choice([1, 40, 1000, 1 << 19])
        keys = [rng.choice([top, 1, rng.randint(0, top)]) if r else 0 for r in rows]
        same = rng.random() < 0.2
        if same:
            keys = [top] * n
            rows = [1] * n
            group = rng.choice([1, 16])
        tokens = max(1, sum(rows)) + rng.choice([0, 0, 20])
        context = rng.choice([0xFFFFFFFF, 32 * top, 200])
        array = ctypes.c_uint32 * n
        index.shares(n, tokens, heads, group, rng.choice([64, 512]), rng.choice([1, max(rows)]), context, array(*rows), array(*keys), o)
        if not o[2]:
            continue
        dealt[max(rows) * group > 64] += 1
        assert o[5] <= o[0] <= o[2] and o[1] <= 128 and o[3] == o[4] <= 1 << 28
        if same and n * heads <= 256 and context >= 32 * top and 256 % (n * heads) == 0 and top == 1 << 19:
            assert o[0] * heads >= 256  # equal lengths fill the chip
    assert min(dealt) > 500
