"""The paged-cache operators and the choice of the next token, as cases that can be timed and compared.

A server's step over several sequences: K and V of the new tokens are normalised, rotated and appended to a paged
cache (fp16, or 4 bits with a scale per 32 values), the new queries attend over their sequences' pages (causal, with
an optional sliding window and a few first tokens that stay visible), and each row of logits gets its penalties,
biases and grammar mask before its largest token is taken.  `run` computes them in their plain form, or, where `own`
is set, through the framework's entry points (include/af.h).

Head layouts, the 1,024-token window, the 32,768-token context, passes of 512 positions and the 262,144-token
vocabulary are those of the framework's own models; the other head widths and the batch sizes are generic.
"""
import ctypes
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
ROPE_CONTEXT = 131072
NO_TOKEN = 0xFFFFFFFF


# ---- the cases ---------------------------------------------------------------------------------

def _append(cache, sequences, new, context, q_heads, kv_heads, width, page, v_norm=False):
    return {"kind": "append", "cache": cache, "sequences": sequences, "new_low": new[0], "new_high": new[1],
            "context_low": context[0], "context_high": context[1], "q_heads": q_heads, "kv_heads": kv_heads,
            "width": width, "page": page, "v_norm": v_norm}


def _attend(cache, sequences, new, context, q_heads, kv_heads, width, page, window=0, sinks=0):
    return {"kind": "attend", "cache": cache, "sequences": sequences, "new_low": new[0], "new_high": new[1],
            "context_low": context[0], "context_high": context[1], "q_heads": q_heads, "kv_heads": kv_heads,
            "width": width, "page": page, "window": window, "sinks": sinks}


def _select(rows, vocabulary, history, biases, allowed):
    return {"kind": "select", "rows": rows, "vocabulary": vocabulary, "history": history, "biases": biases,
            "allowed": allowed}


def listed():
    return [
        # one token of one conversation joins its cache: the smallest call of the path
        dict(_append("f16", 1, (1, 1), (4097, 4097), 16, 8, 256, 16), name="append_1_f16"),
        # a decode step of 64 conversations over a 4-bit cache, and what the cache then holds of it
        dict(_append("q4", 64, (1, 1), (1, 8192), 16, 8, 256, 32), name="append_64_q4"),
        # the prompts of four conversations in one pass, none a multiple of anything
        dict(_append("f16", 4, (301, 611), (301, 2040), 16, 8, 256, 64), name="append_prompts_f16"),
        # one conversation's next token early on: latency
        dict(_attend("f16", 1, (1, 1), (512, 512), 16, 8, 256, 16), name="attend_1_512_f16"),
        # one conversation's next token at the longest context
        dict(_attend("f16", 1, (1, 1), (32768, 32768), 16, 8, 256, 64), name="attend_1_32768_f16"),
        # a decode step of 32 conversations of all lengths
        dict(_attend("f16", 32, (1, 1), (1, 8192), 16, 8, 256, 16), name="attend_32_ragged_f16"),
        # a decode step of 64 long conversations in a sliding-window layer whose first tokens stay visible, 4 bits
        dict(_attend("q4", 64, (1, 1), (100, 16384), 16, 8, 256, 32, 1024, 4), name="attend_64_window_q4"),
        # a decode step of 8 conversations in a global layer: 16 query heads share one 512-wide KV head, 4 bits
        dict(_attend("q4", 8, (1, 1), (2000, 32768), 16, 1, 512, 64), name="attend_8_512wide_q4"),
        # the first pass over one long prompt
        dict(_attend("f16", 1, (512, 512), (512, 512), 16, 8, 256, 64), name="attend_prompt_512_f16"),
        # further turns of four conversations, each a few hundred tokens behind a long history, 4 bits
        dict(_attend("q4", 4, (129, 512), (700, 8192), 16, 8, 256, 64), name="attend_turns_q4"),
        # the next token of one conversation
        dict(_select(1, 262144, 512, 16, 0.5), name="select_1"),
        # the next tokens of 64 conversations, some of them under a narrow grammar
        dict(_select(64, 262144, 2000, 300, 0.1), name="select_64"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "select", "select"])
    if kind == "select":
        vocabulary = _log(rng, 1000, 262144)
        rows = min(_log(rng, 1, 64), (1 << 24) // vocabulary)
        return _select(max(1, rows), vocabulary, _log(rng, 1, 2000), rng.randint(0, 300), rng.choice([0.001, 0.1, 0.5, 1.0]))
    cache, page = rng.choice(["f16", "q4"]), rng.choice([16, 32, 64, 128])
    width = rng.choice([64, 128, 256, 256, 512])
    kv = rng.choice([1, 2, 4, 8]) if width <= 256 else rng.choice([1, 2])
    q = kv * rng.choice([1, 2, 3, 4, 8] if width <= 256 else [1, 4, 16])
    if kind == "append":
        if rng.random() < 0.5:
            return _append(cache, _log(rng, 1, 64), (1, 1), (1, _log(rng, 16, 8192)), q, kv, width, page, rng.random() < 0.3)
        high = _log(rng, 2, 600)
        n = max(1, min(_log(rng, 1, 8), 2048 // high))
        return _append(cache, n, (rng.randint(1, high), high), (high, high + _log(rng, 1, 1500)), q, kv, width, page,
                       rng.random() < 0.3)
    window = rng.choice([0, 0, 0, 512, 1024, 100])
    sinks = rng.choice([0, 1, 4, 37]) if window else 0
    if rng.random() < 0.6:
        high = _log(rng, 1, 32768)
        # no more K and V values than the longest listed batch holds
        n = max(1, min(_log(rng, 1, 64), (1 << 29) // (high * kv * width)))
        return _attend(cache, n, (1, 1), (rng.randint(1, high), high), q, kv, width, page, window, sinks)
    new = _log(rng, 2, 512)
    high = new + _log(rng, 1, 8192)
    n = max(1, min(_log(rng, 1, 8), (1 << 24) * 1024 // (new * high * q * width)))
    return _attend(cache, n, (rng.randint(1, new), new), (new, high), q, kv, width, page, window, sinks)


def _spread(n, low, high, salt):
    """n whole numbers over [low, high] in an order without pattern, both ends among them (for n = 1, high)."""
    order = sorted(range(n), key=lambda i: ((i + 1) * 2654435761 + salt * 40503) % 4294967291)
    return [high if n == 1 else low + (high - low) * k // (n - 1) for k in order]


def _lengths(case):
    """Each sequence's new tokens and its length with them."""
    new = _spread(case["sequences"], case["new_low"], case["new_high"], 1)
    lengths = _spread(case["sequences"], case["context_low"], case["context_high"], 2)
    return new, [max(a, b) for a, b in zip(new, lengths)]


def _scale(case):
    return 1.0 / math.sqrt(case["width"])


# ---- seeded inputs -----------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFFFFFFFFFF)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _page_values(g, case, pages):
    """K or V of all pages as fp16 values, [pages][kv_heads][page][width] (of rounded 4-bit blocks in a 4-bit cache)."""
    shape = (pages, case["kv_heads"], case["page"], case["width"])
    x = _randn(g, *shape)
    if case["cache"] == "f16":
        return x.half()
    code, d = _quantise(x.reshape(-1, 32))
    return _pack(code.reshape(shape), d.reshape(*shape[:3], -1))


def _inputs(case, seed):
    """The inputs as GPU tensors, the same whatever computes on them."""
    g = _generator(seed)
    if case["kind"] == "select":
        rows, vocab, biases = case["rows"], case["vocabulary"], case["biases"]
        t = {"logits": 3.0 * _randn(g, rows, vocab)}
        # the ids so far: a few common tokens many times, others once; rows of different lengths
        h = torch.rand(rows, case["history"], generator=g, device=DEV).pow(4.0).mul(vocab).long().clamp(max=vocab - 1)
        t["history"] = h.int()
        t["history_len"] = torch.randint(0, case["history"] + 1, (rows,), generator=g, device=DEV).int()
        u = torch.rand(rows, 3, generator=g, device=DEV)
        t["penalties"] = u * torch.tensor([0.5, 1.0, 1.0], device=DEV) + torch.tensor([1.0, 0.0, 0.0], device=DEV)
        t["bias_ids"] = torch.randint(0, vocab, (rows, max(1, biases)), generator=g, device=DEV).int()
        t["bias_values"] = 4.0 * _randn(g, rows, max(1, biases))
        t["bias_len"] = torch.randint(0, biases + 1, (rows,), generator=g, device=DEV).int()
        words = (vocab + 31) // 32
        allow = torch.rand(rows, words * 32, generator=g, device=DEV) < case["allowed"]
        bit = torch.ones((), dtype=torch.int64, device=DEV) << torch.arange(32, device=DEV)
        t["mask"] = (allow.reshape(rows, words, 32).long() * bit).sum(-1).int()
        return t
    new, lengths = _lengths(case)
    kv, w, page = case["kv_heads"], case["width"], case["page"]
    tokens, entries = sum(new), [-(-n // page) for n in lengths]
    pages = sum(entries) + 3
    t = {"starts": torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEV),
         "lengths": torch.tensor(lengths, dtype=torch.int32, device=DEV)}
    # the sequences' pages lie anywhere in the pool; entries behind a sequence's last page are no page
    order = torch.randperm(pages, generator=g, device=DEV).int()
    width = max(entries)
    first = torch.tensor([sum(entries[:i]) for i in range(len(entries))], device=DEV)[:, None]
    at = torch.arange(width, device=DEV)[None]
    held = at < torch.tensor(entries, device=DEV)[:, None]
    t["table"] = torch.where(held, order[(first + at).clamp(max=pages - 1)], torch.full((), -1, dtype=torch.int32, device=DEV))
    t["table"] = t["table"].contiguous()
    t["k_pages"], t["v_pages"] = _page_values(g, case, pages), _page_values(g, case, pages)
    if case["kind"] == "append":
        t["q"], t["k"], t["v"] = (_randn(g, tokens, h, w) for h in (case["q_heads"], kv, kv))
        t["q_norm"], t["k_norm"] = 1.0 + 0.1 * _randn(g, w), 1.0 + 0.1 * _randn(g, w)
    else:
        t["q"] = 2.0 * _randn(g, tokens, case["q_heads"], w)
    return t


def _factors(width):
    """RoPE frequency divisors: a global 512-wide layer turns only its first 64 pairs."""
    f = [1.0] * (width // 2)
    return [1.0] * 64 + [1e30] * (width // 2 - 64) if width == 512 else f


def prepare(case, seed):
    t = _inputs(case, seed)
    s = {"case": case, **t}
    if case["kind"] == "select":
        s["out"] = torch.empty_like(t["logits"])
        s["result"] = torch.empty(case["rows"], 2, dtype=torch.int32, device=DEV)
    elif case["kind"] == "append":
        tokens, kv, w = t["k"].shape
        s["q_out"] = torch.empty_like(t["q"])
        s["values"] = [torch.empty(tokens, kv, w, dtype=torch.float16, device=DEV) for _ in range(2)]
    else:
        s["out"] = torch.empty_like(t["q"])
    if own:
        _bind(s)
    return s


# ---- the framework's calls -----------------------------------------------------------------------

class _Handle:
    """A handle of the library, freed with the state that holds it."""

    def __init__(self, h, free):
        self.h, self.free = h, free

    def __del__(self):
        self.free(self.h)


def _bind(s):
    """What a program keeps between calls: the argument structs, the RoPE handle and the workspace."""
    from adaforge_amd import _native as N
    case, lib = s["case"], N.lib()
    p = lambda n: s[n].data_ptr()  # noqa: E731
    s["native"], s["device"] = N, torch.cuda.current_device()
    size = N.sz()
    if case["kind"] == "select":
        a = N.LogitsArgs(p("logits"), case["vocabulary"], p("out"), case["vocabulary"], case["rows"], case["vocabulary"],
                         p("penalties"), p("history"), s["history"].shape[1], p("history_len"), p("bias_ids"),
                         p("bias_values"), s["bias_ids"].shape[1], p("bias_len"), p("mask"), s["mask"].shape[1], p("result"),
                         None)
        N.check(lib.af_logits_select_workspace(ctypes.byref(a), ctypes.byref(size)))
    else:
        tokens = s["q"].shape[0]
        pages = N.KvPages(p("k_pages"), p("v_pages"), N.AF_KV_F16 if case["cache"] == "f16" else N.AF_KV_Q4,
                          s["k_pages"].shape[0], case["page"], case["kv_heads"], case["width"])
        batch = N.KvBatch(p("starts"), p("lengths"), p("table"), s["table"].shape[1], case["sequences"], tokens)
        qd, kd = case["q_heads"] * case["width"], case["kv_heads"] * case["width"]
        if case["kind"] == "append":
            factors = (ctypes.c_float * (case["width"] // 2))(*_factors(case["width"]))
            h = N.P()
            N.check(lib.af_rope_create(ctypes.byref(N.RopeDesc(case["width"], 1e6, factors, ROPE_CONTEXT)), ctypes.byref(h)))
            s["rope"] = _Handle(h, lib.af_rope_free)
            s["args"] = N.KvAppendArgs(p("q"), qd, p("k"), kd, p("v"), kd, p("q_norm"), p("k_norm"), EPS, EPS, EPS,
                                       1 if case["v_norm"] else 0, h, case["q_heads"], p("q_out"), qd, pages, batch)
            return
        a = N.PagedAttentionArgs(p("q"), qd, p("out"), qd,
                                 N.AttentionConfigDesc(case["q_heads"], case["kv_heads"], case["width"], case["window"],
                                                       _scale(case)),
                                 case["sinks"], pages, batch, max(_lengths(case)[0]), max(_lengths(case)[1]), None)
        N.check(lib.af_paged_attention_workspace(ctypes.byref(a), ctypes.byref(size)))
    h = N.P()
    N.check(lib.af_workspace_create(size.value, ctypes.byref(h)))
    s["workspace"], a.workspace = _Handle(h, lib.af_workspace_free), h
    s["args"] = a


def _run_own(s):
    N, case, kind = s["native"], s["case"], s["case"]["kind"]
    # (the number alone: a stream object takes 2.7 us, as long as the shortest pass)
    lib, stream = N.lib(), torch._C._cuda_getCurrentRawStream(s["device"])
    if kind == "select":
        N.check(lib.af_logits_select(ctypes.byref(s["args"]), stream))
        return {"logits": s["out"], "result": s["result"]}
    if kind == "attend":
        N.check(lib.af_paged_attention(ctypes.byref(s["args"]), stream))
        return s["out"]
    N.check(lib.af_kv_append(ctypes.byref(s["args"]), stream))
    if case["cache"] == "f16":
        return {"q": s["q_out"], "k": s["k_pages"], "v": s["v_pages"]}
    k, v = s["values"]
    a = s["args"]
    N.check(lib.af_kv_read(ctypes.byref(a.pages), ctypes.byref(a.batch), k.data_ptr(), v.data_ptr(), stream))
    return {"q": s["q_out"], "k": k, "v": v}


# ---- the plain form ------------------------------------------------------------------------------
#
# A 4-bit page holds, for each KV head, the codes of its tokens and then their scales: a block of 32 values has the
# fp16 scale d = -m / 8, m its value of largest magnitude (the positive one of two), and codes n = rint(x / d) + 8 in
# 0 .. 15, which stand for the fp16 value of d (n - 8).  Eight codes make a 32-bit word: values 2 i and 2 i + 1 at
# bits 4 i and 16 + 4 i.

def _quantise(x):
    """Codes [n][32] and scales [n] of blocks x [n][32] (32 bits)."""
    high, low = x.amax(1), x.amin(1)
    d = (torch.where(high >= -low, high, low) / -8.0).half()
    ratio = x.double() / d.double()[:, None]
    code = torch.where(d[:, None] == 0, torch.full_like(ratio, 8.0), torch.round(ratio) + 8.0).clamp(0, 15)
    return code.to(torch.uint8), d


def _words(code):
    """Packed bytes [..., width / 2] of codes [..., width]."""
    shift = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device=DEV)
    word = (code.reshape(*code.shape[:-1], -1, 8).long() << shift).sum(-1)
    return (word & 0xFFFFFFFF).to(torch.uint32).view(torch.uint8)


def _pack(code, d):
    """Page bytes [pages][kv_heads][page * width * 9 / 16]."""
    n, kv = code.shape[:2]
    return torch.cat([_words(code).reshape(n, kv, -1), d.contiguous().view(torch.uint8).reshape(n, kv, -1)], 2)


def _planes(pages, page, width):
    """Views of the codes' bytes [pages][kv_heads][page][width / 2] and the scales [pages][kv_heads][page][width / 32]."""
    n, kv, cut = pages.shape[0], pages.shape[1], page * width // 2
    return (pages[:, :, :cut].unflatten(2, (page, width // 2)),
            pages[:, :, cut:].view(torch.float16).unflatten(2, (page, width // 32)))


def _codes(words):
    """Codes [..., width] of packed bytes [..., width / 2]."""
    shift = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device=DEV)
    return ((words.contiguous().view(torch.int32).unsqueeze(-1) >> shift) & 15).flatten(-2)


def _stands_for(code, d):
    """The fp16 values of codes [..., width] under scales [..., width / 32]."""
    v = (code.float() - 8.0).unflatten(-1, (-1, 32)) * d.float().unsqueeze(-1)
    return v.half().flatten(-2)


def _held(case, pages, at):
    """The 32-bit values of pages `at` [sequences][n], as [sequences][kv_heads][n * page][width]."""
    if case["cache"] == "f16":
        x = pages[at]
    else:
        words, d = _planes(pages, case["page"], case["width"])
        x = _stands_for(_codes(words[at]), d[at])
    return x.transpose(1, 2).flatten(2, 3).float()


def _places(s):
    """Each token's sequence, position, page and slot."""
    case, starts = s["case"], s["starts"].long()
    token = torch.arange(s["q"].shape[0], device=DEV)
    seq = torch.searchsorted(starts, token, right=True) - 1
    pos = s["lengths"].long()[seq] - starts[seq + 1] + token
    page = s["table"].long()[seq, pos // case["page"]]
    return seq, pos, page, pos % case["page"]


def _normed(x, w):
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * r if w is None else x * r * w.double()


def _rotated(x, pos):
    half = x.shape[-1] // 2
    i = torch.arange(half, device=DEV, dtype=torch.float64)
    f = 1e6 ** (-i / half) / torch.tensor(_factors(2 * half), dtype=torch.float32, device=DEV).double()
    a = pos.double()[:, None, None] * f
    sin, cos = torch.sin(a), torch.cos(a)
    u, v = x[..., :half], x[..., half:]
    return torch.cat([u * cos - v * sin, u * sin + v * cos], -1)


def _plain_append(s):
    # 64 bits up to the one rounding to 32: angles of far positions, and values next to a code's border
    case = s["case"]
    _, pos, page, slot = _places(s)
    q = _rotated(_normed(s["q"].double(), s["q_norm"]), pos).float()
    k = _rotated(_normed(s["k"].double(), s["k_norm"]), pos).float()
    v = _normed(s["v"].double(), None).float() if case["v_norm"] else s["v"]
    if case["cache"] == "f16":
        s["k_pages"][page, :, slot] = k.half()
        s["v_pages"][page, :, slot] = v.half()
        return {"q": q, "k": s["k_pages"], "v": s["v_pages"]}
    return {"q": q, "k": _store4(case, s["k_pages"], k, page, slot), "v": _store4(case, s["v_pages"], v, page, slot)}


def _store4(case, pages, x, page, slot):
    code, d = _quantise(x.reshape(-1, 32))
    code, d = code.reshape(x.shape), d.reshape(*x.shape[:2], -1)
    words, scales = _planes(pages, case["page"], case["width"])
    words[page, :, slot] = _words(code)
    scales[page, :, slot] = d
    return _stands_for(code, d)


def _plain_attend(s):
    case = s["case"]
    S, qh, kv, w = case["sequences"], case["q_heads"], case["kv_heads"], case["width"]
    starts, lengths = s["starts"].long(), s["lengths"].long()
    new = starts[1:] - starts[:-1]
    most = max(_lengths(case)[0])
    # the pages that any of a sequence's queries sees: those of the first tokens, then from the window's first on
    P, column = case["page"], torch.arange(s["table"].shape[1], device=DEV)[None]
    if case["window"]:
        first = -(-case["sinks"] // P)
        start = ((lengths - new + 1 - case["window"]).clamp(min=0) // P).clamp(min=first)[:, None]
        column = torch.arange(first + (case["window"] + most) // P + 2, device=DEV)[None]
        column = torch.where(column < first, column, start + column - first)
    at = torch.gather(s["table"].long(), 1, column.clamp(max=s["table"].shape[1] - 1).expand(S, -1)).clamp(min=0)
    k, v = _held(case, s["k_pages"], at), _held(case, s["v_pages"], at)
    key = (column[:, :, None] * P + torch.arange(P, device=DEV)).flatten(1).expand(S, -1)
    i = torch.arange(most, device=DEV)
    valid = i[None] < new[:, None]
    token = (starts[:-1, None] + i[None]).clamp(max=s["q"].shape[0] - 1)
    pos = (lengths - new)[:, None] + i[None]
    # queries of a KV head's group together: [sequences][kv_heads][most * group][width]
    q = s["q"][token].reshape(S, most, kv, qh // kv, w).permute(0, 2, 1, 3, 4).reshape(S, kv, -1, w)
    seen = key[:, None] <= pos[:, :, None]
    if case["window"]:
        seen &= (key[:, None] > pos[:, :, None] - case["window"]) | (key[:, None] < case["sinks"])
    v = torch.where((key < lengths[:, None])[:, None, :, None], v, torch.zeros((), device=DEV))
    score = torch.matmul(q, k.transpose(2, 3)).mul_(_scale(case)).unflatten(2, (most, -1))
    score = score.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (most, -1)) / torch.where(total == 0, torch.ones_like(total), total)
    s["out"][token[valid]] = o.permute(0, 2, 1, 3, 4).reshape(S, most, qh, w)[valid]
    return s["out"]


def _plain_select(s):
    case, x = s["case"], s["logits"]
    rows, vocab = x.shape
    row = torch.arange(rows, device=DEV)[:, None]
    i = torch.arange(s["history"].shape[1], device=DEV)[None]
    count = torch.zeros(rows, vocab, dtype=torch.int32, device=DEV)
    count.scatter_add_(1, s["history"].long(), (i < s["history_len"][:, None]).int())
    # of an id's biases the last counts
    j = torch.arange(s["bias_ids"].shape[1], device=DEV)[None]
    last = torch.zeros(rows, vocab, dtype=torch.int64, device=DEV)
    last.scatter_reduce_(1, s["bias_ids"].long(), torch.where(j < s["bias_len"][:, None], j + 1, 0), "amax")
    bias = torch.where(last > 0, s["bias_values"][row, (last - 1).clamp(min=0)], torch.zeros((), device=DEV))
    # 64 bits up to the one rounding: equal values stay equal, and the order of neighbours holds
    rep, presence, frequency = (s["penalties"][:, c:c + 1].double() for c in range(3))
    y = x.double()
    y = torch.where(count > 0, torch.where(y > 0, y / rep, y * rep) - (frequency * count + presence), y)
    y = (y + bias.double()).float()
    bit = torch.arange(vocab, device=DEV)
    allow = (s["mask"][:, bit // 32] >> (bit % 32).int()) & 1
    y = torch.where(allow == 1, y, torch.full((), -math.inf, device=DEV))
    top = y.amax(1, keepdim=True)
    best = torch.where(y == top, bit[None], vocab).amin(1)
    best = torch.where(top[:, 0] == -math.inf, -1, best)  # no token: all bits set
    bad = (torch.isnan(y) | (y == math.inf)).any(1)
    return {"logits": y, "result": torch.stack([best, bad.long()], 1).int()}


def run(s):
    if own:
        return _run_own(s)
    return {"append": _plain_append, "attend": _plain_attend, "select": _plain_select}[s["case"]["kind"]](s)


# ---- what a pass cannot do without ---------------------------------------------------------------

def _row_bytes(case):
    """Bytes of one token's K (V alike) in the cache, all heads."""
    return case["kv_heads"] * case["width"] * (16 if case["cache"] == "f16" else 9) // (8 if case["cache"] == "f16" else 16)


def _visible(case, pos):
    """How many keys position pos sees."""
    if not case["window"]:
        return pos + 1
    first = max(0, pos + 1 - case["window"])
    return pos + 1 - first + min(first, case["sinks"])


def work(case):
    if case["kind"] == "select":
        r, v = case["rows"], case["vocabulary"]
        return {"bytes": r * (8 * v + v // 8 + 4 * case["history"] // 2 + 4 * case["biases"]), "flops": r * v}
    new, lengths = _lengths(case)
    qd, tokens = case["q_heads"] * case["width"], sum(new)
    if case["kind"] == "append":
        kd = case["kv_heads"] * case["width"]
        back = 0 if case["cache"] == "f16" else 2 * _row_bytes(case) + 4 * kd  # the values read back
        return {"bytes": tokens * (8 * qd + 8 * kd + 2 * _row_bytes(case) + back), "flops": 10 * tokens * (qd + 2 * kd)}
    keys = pairs = 0
    for n, length in zip(new, lengths):
        first = max(0, length - n + 1 - case["window"]) if case["window"] else 0
        keys += length - first + min(first, case["sinks"])
        pairs += sum(_visible(case, p) for p in range(length - n, length))
    return {"bytes": 2 * keys * _row_bytes(case) + 8 * tokens * qd, "flops": 4 * pairs * qd}


# ---- the 64-bit answers, written apart from the plain form ------------------------------------------

def _exact_blocks(x):
    """The values that 4-bit blocks of x (64 bits, rounded to 32 first) stand for."""
    b = x.float().double().reshape(-1, 32)
    big = b.abs().amax(1)
    m = torch.where((b == big[:, None]).any(1), big, -big)
    d = (m.float() / -8).half().double()[:, None]
    n = torch.where(d == 0, torch.zeros_like(b), torch.round(b / d).clamp(-8, 7))
    return (n * d).float().half().double().reshape(x.shape)


def _unpack(pages, case):
    """64-bit values [pages][kv_heads][page][width] of a pool's bytes."""
    if case["cache"] == "f16":
        return pages.double()
    n, kv, P, w = pages.shape[0], case["kv_heads"], case["page"], case["width"]
    b = pages[:, :, :P * w // 2].reshape(n, kv, P, w // 8, 4)
    d = pages[:, :, P * w // 2:].contiguous().view(torch.float16).reshape(n, kv, P, w // 32)
    # byte j of a word holds values 2 (j % 2 * 2) + (j >= 2) and the next pair's
    low, high = (b & 15).double() - 8, (b >> 4).double() - 8
    v = torch.stack([low[..., 0], low[..., 2], high[..., 0], high[..., 2],
                     low[..., 1], low[..., 3], high[..., 1], high[..., 3]], -1).reshape(n, kv, P, w // 32, 32)
    return (v * d.double()[..., None]).float().half().double().reshape(n, kv, P, w)


def _exact_append(case, t):
    new, lengths = _lengths(case)
    P, w, half = case["page"], case["width"], case["width"] // 2
    pos = torch.cat([torch.arange(n - m, n, device=DEV) for m, n in zip(new, lengths)])
    turn = torch.pow(torch.tensor(1e6, dtype=torch.float64, device=DEV), torch.arange(half, device=DEV).double() * (-2.0 / w))
    angle = torch.outer(pos.double(), turn / torch.tensor(_factors(w), device=DEV, dtype=torch.float32).double())
    wheel = torch.polar(torch.ones_like(angle), angle)[:, None]

    def turned(x, weight):
        x = x.double()
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * weight.double()
        z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * wheel
        return torch.cat([z.real, z.imag], -1)

    q, k, v = turned(t["q"], t["q_norm"]), turned(t["k"], t["k_norm"]), t["v"].double()
    if case["v_norm"]:
        v = v / torch.sqrt(v.pow(2).mean(-1, keepdim=True) + EPS)
    if case["cache"] == "q4":
        return {"q": q, "k": _exact_blocks(k), "v": _exact_blocks(v)}
    kp, vp = t["k_pages"].double(), t["v_pages"].double()
    i = 0
    for s, (m, n) in enumerate(zip(new, lengths)):
        p = torch.arange(n - m, n, device=DEV)
        page = t["table"][s].long()[p // P]
        kp[page, :, p % P], vp[page, :, p % P] = k[i:i + m], v[i:i + m]
        i += m
    return {"q": q, "k": kp, "v": vp}


def _exact_attend(case, t):
    new, lengths = _lengths(case)
    group, P = case["q_heads"] // case["kv_heads"], case["page"]
    out, i = torch.zeros(t["q"].shape, dtype=torch.float64, device=DEV), 0
    for s, (m, n) in enumerate(zip(new, lengths)):
        pages = t["table"][s, :-(-n // P)].long()
        rows = lambda x: _unpack(x[pages], case).permute(1, 0, 2, 3).reshape(case["kv_heads"], -1, case["width"])[:, :n]  # noqa: E731
        k, v = rows(t["k_pages"]), rows(t["v_pages"])
        p = torch.arange(n - m, n, device=DEV)[:, None]
        key = torch.arange(n, device=DEV)[None]
        hidden = key > p
        if case["window"]:
            hidden |= (p - key >= case["window"]) & (key >= case["sinks"])
        for h in range(case["q_heads"]):
            a = t["q"][i:i + m, h].double() @ k[h // group].t().contiguous() * _scale(case)
            out[i:i + m, h] = torch.softmax(a.masked_fill(hidden, -math.inf), -1) @ v[h // group]
        i += m
    return out


def _exact_select(case, t):
    y = t["logits"].double()
    for r in range(case["rows"]):
        rep, presence, frequency = t["penalties"][r].double().tolist()
        ids, n = torch.unique(t["history"][r, :int(t["history_len"][r])].long(), return_counts=True)
        x = y[r, ids]
        y[r, ids] = torch.where(x > 0, x / rep, x * rep) - presence - frequency * n
        at = {}
        for i, b in zip(t["bias_ids"][r, :int(t["bias_len"][r])].tolist(), t["bias_values"][r].tolist()):
            at[i] = b
        if at:
            y[r, list(at)] += torch.tensor(list(at.values()), dtype=torch.float64, device=DEV)
        words = t["mask"][r].long()[:, None] >> torch.arange(32, device=DEV)[None]
        y[r, (words & 1).reshape(-1)[:case["vocabulary"]] == 0] = -math.inf
    return {"logits": y, "result": None}


def exact(case, seed):
    return {"append": _exact_append, "attend": _exact_attend, "select": _exact_select}[case["kind"]](case, _inputs(case, seed))
