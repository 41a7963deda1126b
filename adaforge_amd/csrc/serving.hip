// Host side of the operators over several sequences (include/af.h): workspaces, RoPE frequencies, checks of arguments
// before any GPU work, launches.  No call here allocates, waits or changes the current device but the create and
// free functions, so all of them can be captured into graphs.
#include <hip/hip_runtime.h>

#include <atomic>
#include <cmath>
#include <cstring>
#include <new>
#include <string>
#include <vector>

#include "../../include/af.h"
#include "af_internal.h"
#include "paged.h"

using namespace af;

struct af_workspace {
    void* p = nullptr;
    size_t bytes = 0;
    int device = 0;
};

struct af_rope {
    uint64_t* turns = nullptr;
    uint32_t width = 0;
    int device = 0;
};

namespace {

// An entry point's body: what is thrown inside (a message's memory) does not leave it.
template <typename F>
int guarded(F f) noexcept {
    try {
        return f();
    } catch (...) {
        return AF_ERR_DEVICE;
    }
}

int fail(int code, const char* msg) { return set_error(code, msg); }
int fail(hipError_t e, const char* what) { return set_error(AF_ERR_DEVICE, std::string(what) + ": " + hipGetErrorString(e)); }

// The current device, which has to be a gfx950.
int current_device(int* out) {
    int n = 0, dev = 0;
    if (hipGetDeviceCount(&n) != hipSuccess || n < 1) return fail(AF_ERR_NO_DEVICE, "no HIP device");
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return fail(e, "current device");
    static std::atomic<uint64_t> known{0};  // devices already seen to be gfx950 (asking takes about 0.1 ms)
    if (dev >= 64 || !(known.load() >> dev & 1)) {
        hipDeviceProp_t p;
        if ((e = hipGetDeviceProperties(&p, dev)) != hipSuccess) return fail(e, "device properties");
        if (std::strncmp(p.gcnArchName, "gfx950", 6) != 0)
            return set_error(AF_ERR_NO_DEVICE, std::string("gfx950 (MI355X) required, found ") + p.gcnArchName);
        if (dev < 64) known.fetch_or(1ull << dev);
    }
    *out = dev;
    return AF_OK;
}

// Whether `stream` runs on `device`, where the handle that the call uses lives.
int check_stream(void* stream, int device, const char* what) {
    int dev = -1;
    hipDevice_t d;
    const hipError_t e = stream ? hipStreamGetDevice((hipStream_t)stream, &d) : hipGetDevice(&dev);
    if (e != hipSuccess) return fail(e, "stream's device");
    if (stream) dev = (int)d;
    if (dev != device) return set_error(AF_ERR_INVALID, std::string(what) + " lives on another device than the stream");
    return AF_OK;
}

bool aligned(const void* p) { return (uintptr_t)p % 16 == 0; }

bool page_size(uint32_t page) { return page >= 16 && page <= 256 && (page & (page - 1)) == 0; }

int check_pages(const af_kv_pages& p) {
    if (!p.k || !p.v) return fail(AF_ERR_INVALID, "null cache pages");
    if (!aligned(p.k) || !aligned(p.v)) return fail(AF_ERR_INVALID, "cache pages must be 16-byte aligned");
    if (p.pages == 0 || p.pages > 0x7FFFFFFFu) return fail(AF_ERR_INVALID, "invalid number of cache pages");
    if (!af_kv_page_bytes(p.type, p.page, p.kv_heads, p.width))
        return fail(AF_ERR_INVALID, "unsupported cache layout (type, 16 to 256 tokens a page, 1 to 1024 heads, width 64, 128, 256 or 512)");
    return AF_OK;
}

int check_batch(const af_kv_batch& b, uint32_t page) {
    if (!b.starts || !b.lengths || !b.table) return fail(AF_ERR_INVALID, "null batch array");
    if (b.sequences == 0 || b.sequences > AF_MAX_SEQUENCES) return fail(AF_ERR_INVALID, "invalid number of sequences");
    if (b.tokens == 0 || b.tokens > AF_MAX_BATCH_TOKENS) return fail(AF_ERR_INVALID, "invalid number of batch tokens");
    if (b.table_stride == 0 || b.table_stride > AF_MAX_POSITIONS / page)
        return fail(AF_ERR_INVALID, "page table rows must hold 1 to 16777216 positions");
    return AF_OK;
}

int check_rows(const void* p, uint32_t stride, uint64_t row, const char* what) {
    if (!p) return set_error(AF_ERR_INVALID, std::string("null ") + what);
    if (!aligned(p) || stride % 4 != 0)
        return set_error(AF_ERR_INVALID, std::string(what) + " must be 16-byte aligned, its stride a multiple of 4");
    if (stride < row) return set_error(AF_ERR_INVALID, std::string(what) + " rows overlap: the stride is less than a row");
    return AF_OK;
}

PagedBatch batch_view(const af_kv_batch& b, const af_kv_pages& p) {
    return {b.starts, b.lengths, b.table, b.table_stride, b.sequences, b.tokens, p.pages, (uint32_t)__builtin_ctz(p.page)};
}

int check_workspace(const af_workspace* w, size_t need, void* stream) {
    if (!w) return fail(AF_ERR_INVALID, "null workspace");
    if (w->bytes < need)
        return set_error(AF_ERR_INVALID, "the workspace has " + std::to_string(w->bytes) + " bytes, the call needs " + std::to_string(need));
    return check_stream(stream, w->device, "the workspace");
}

bool positive(float e) { return std::isfinite(e) && e > 0.0f; }

// What the sizes of an attention call have to be, apart from its pointers.
int check_attention_sizes(const af_paged_attention_args& a) {
    const af_attention_config& c = a.config;
    if (c.q_heads == 0 || c.kv_heads == 0 || c.q_heads % c.kv_heads != 0 || c.q_heads > AF_MAX_HEADS || !positive(c.scale))
        return fail(AF_ERR_INVALID, "invalid attention configuration");
    if (c.kv_heads != a.pages.kv_heads || c.width != a.pages.width)
        return fail(AF_ERR_INVALID, "the attention's KV heads or width differ from the cache's");
    if (!af_kv_page_bytes(a.pages.type, a.pages.page, a.pages.kv_heads, a.pages.width))
        return fail(AF_ERR_INVALID, "unsupported cache layout (type, 16 to 256 tokens a page, 1 to 1024 heads, width 64, 128, 256 or 512)");
    if (a.batch.sequences == 0 || a.batch.sequences > AF_MAX_SEQUENCES || a.batch.tokens == 0 || a.batch.tokens > AF_MAX_BATCH_TOKENS)
        return fail(AF_ERR_INVALID, "invalid number of sequences or batch tokens");
    if ((uint64_t)a.batch.sequences * c.kv_heads > 1u << 22) return fail(AF_ERR_INVALID, "sequences times KV heads above 4194304");
    return AF_OK;
}

AttnShape shape_of(const af_paged_attention_args& a) {
    const af_attention_config& c = a.config;
    return {a.batch.sequences, a.batch.tokens,    c.kv_heads,        c.q_heads / c.kv_heads, c.width, c.window, a.sinks,
            a.longest_query,   a.longest_context, least(a.batch.table_stride, AF_MAX_POSITIONS / a.pages.page) * a.pages.page,
            a.pages.type == AF_KV_Q4};
}

}  // namespace

extern "C" {

int af_workspace_create(size_t bytes, af_workspace** out) {
    return guarded([&]() -> int {
        if (!out) return fail(AF_ERR_INVALID, "null output");
        *out = nullptr;
        int dev = 0;
        const int rc = current_device(&dev);
        if (rc) return rc;
        af_workspace* w = new (std::nothrow) af_workspace;
        if (!w) return fail(AF_ERR_DEVICE, "out of host memory");
        w->bytes = bytes < kTicketBytes ? kTicketBytes : bytes;
        w->device = dev;
        hipError_t e = hipMalloc(&w->p, w->bytes);
        if (e == hipSuccess) e = hipMemset(w->p, 0, kTicketBytes);
        if (e == hipSuccess) e = hipDeviceSynchronize();
        if (e != hipSuccess) {
            af_workspace_free(w);
            return fail(e, "workspace");
        }
        *out = w;
        return AF_OK;
    });
}

void af_workspace_free(af_workspace* w) {
    if (!w) return;
    if (w->p) (void)hipFree(w->p);
    delete w;
}

int af_rope_create(const af_rope_params* p, af_rope** out) {
    return guarded([&]() -> int {
        if (!out) return fail(AF_ERR_INVALID, "null output");
        *out = nullptr;
        if (!p || p->width == 0 || p->width > 65536 || p->width % 2 != 0 || !p->factors || !std::isfinite(p->base) ||
            p->base <= 1.0 || p->context == 0)
            return fail(AF_ERR_INVALID, "invalid RoPE parameters");
        for (uint32_t i = 0; i < p->width / 2; ++i)
            if (!positive(p->factors[i])) return fail(AF_ERR_INVALID, "invalid RoPE parameters");
        int dev = 0;
        const int rc = current_device(&dev);
        if (rc) return rc;
        af_rope* r = new (std::nothrow) af_rope;
        uint64_t* host = new (std::nothrow) uint64_t[p->width / 2];
        if (!r || !host) {
            delete r;
            delete[] host;
            return fail(AF_ERR_DEVICE, "out of host memory");
        }
        for (uint32_t i = 0; i < p->width / 2; ++i) {
            const long double turn = powl((long double)p->base, -2.0L * i / p->width) / (long double)p->factors[i] /
                                     6.283185307179586476925286766559005768L;
            const long double f = rintl(ldexpl(turn - floorl(turn), 64));
            host[i] = f >= 18446744073709551616.0L ? 0 : (uint64_t)f;
        }
        r->width = p->width;
        r->device = dev;
        hipError_t e = hipMalloc((void**)&r->turns, (size_t)p->width / 2 * 8);
        if (e == hipSuccess) e = hipMemcpy(r->turns, host, (size_t)p->width / 2 * 8, hipMemcpyHostToDevice);
        delete[] host;
        if (e != hipSuccess) {
            af_rope_free(r);
            return fail(e, "RoPE frequencies");
        }
        *out = r;
        return AF_OK;
    });
}

void af_rope_free(af_rope* r) {
    if (!r) return;
    if (r->turns) (void)hipFree(r->turns);
    delete r;
}

size_t af_kv_page_bytes(uint32_t type, uint32_t page, uint32_t kv_heads, uint32_t width) {
    if ((type != AF_KV_F16 && type != AF_KV_Q4) || !page_size(page) || kv_heads == 0 || kv_heads > AF_MAX_HEADS ||
        (width != 64 && width != 128 && width != 256 && width != 512))
        return 0;
    return (size_t)kv_heads * page_part_bytes(type == AF_KV_Q4, page, width);
}

int af_kv_append(const af_kv_append_args* p, void* stream) {
    return guarded([&]() -> int {
        if (!p) return fail(AF_ERR_INVALID, "null append arguments");
        int rc;
        if ((rc = check_pages(p->pages))) return rc;
        if ((rc = check_batch(p->batch, p->pages.page))) return rc;
        const uint64_t w = p->pages.width, kd = w * p->pages.kv_heads, qd = w * p->q_heads;
        if ((rc = check_rows(p->k, p->k_stride, kd, "k"))) return rc;
        if ((rc = check_rows(p->v, p->v_stride, kd, "v"))) return rc;
        if ((p->q != nullptr) != (p->q_heads != 0) || p->q_heads > AF_MAX_HEADS)
            return fail(AF_ERR_INVALID, "q and 1 to 1024 query heads go together");
        if (p->q) {
            if ((rc = check_rows(p->q, p->q_stride, qd, "q"))) return rc;
            if ((rc = check_rows(p->q_out, p->q_out_stride, qd, "q_out"))) return rc;
            if (p->q_out == p->q && p->q_out_stride != p->q_stride)
                return fail(AF_ERR_INVALID, "q_out in place of q must have its stride");
        }
        if ((p->q && p->q_norm && !positive(p->q_eps)) || (p->k_norm && !positive(p->k_eps)) || (p->v_norm && !positive(p->v_eps)))
            return fail(AF_ERR_INVALID, "epsilon must be finite and positive");
        if (p->rope) {
            if (p->rope->width != w) return fail(AF_ERR_INVALID, "RoPE width differs from head width");
            if ((rc = check_stream(stream, p->rope->device, "the RoPE handle"))) return rc;
        }
        KvAppend a{};
        a.q = p->q;
        a.k = p->k;
        a.v = p->v;
        a.q_stride = p->q_stride;
        a.k_stride = p->k_stride;
        a.v_stride = p->v_stride;
        a.q_norm = p->q_norm;
        a.k_norm = p->k_norm;
        a.q_eps = p->q_eps;
        a.k_eps = p->k_eps;
        a.v_eps = p->v_eps;
        a.v_norm = p->v_norm != 0;
        a.turns = p->rope ? p->rope->turns : nullptr;
        a.q_heads = p->q_heads;
        a.kv_heads = p->pages.kv_heads;
        a.q_out = p->q_out;
        a.q_out_stride = p->q_out_stride;
        a.k_pages = (uint8_t*)p->pages.k;
        a.v_pages = (uint8_t*)p->pages.v;
        a.b = batch_view(p->batch, p->pages);
        const hipError_t e = launch_kv_append(a, p->pages.width, p->pages.type == AF_KV_Q4, (hipStream_t)stream);
        return e == hipSuccess ? AF_OK : fail(e, "KV append launch");
    });
}

int af_kv_read(const af_kv_pages* pages, const af_kv_batch* batch, uint16_t* k, uint16_t* v, void* stream) {
    return guarded([&]() -> int {
        if (!pages || !batch || !k || !v) return fail(AF_ERR_INVALID, "null argument");
        int rc;
        if ((rc = check_pages(*pages))) return rc;
        if ((rc = check_batch(*batch, pages->page))) return rc;
        if (!aligned(k) || !aligned(v)) return fail(AF_ERR_INVALID, "k and v must be 16-byte aligned");
        const hipError_t e = launch_kv_read((const uint8_t*)pages->k, (const uint8_t*)pages->v, batch_view(*batch, *pages),
                                            pages->kv_heads, pages->width, pages->type == AF_KV_Q4, k, v, (hipStream_t)stream);
        return e == hipSuccess ? AF_OK : fail(e, "KV read launch");
    });
}

int af_paged_attention_workspace(const af_paged_attention_args* p, size_t* bytes) {
    return guarded([&]() -> int {
        if (!p || !bytes) return fail(AF_ERR_INVALID, "null argument");
        const int rc = check_attention_sizes(*p);
        if (rc) return rc;
        *bytes = kTicketBytes + attn_plan(shape_of(*p)).part_bytes;
        return AF_OK;
    });
}

int af_paged_attention(const af_paged_attention_args* p, void* stream) {
    return guarded([&]() -> int {
        size_t need = 0;
        int rc = af_paged_attention_workspace(p, &need);
        if (rc) return rc;
        if ((rc = check_pages(p->pages))) return rc;
        if ((rc = check_batch(p->batch, p->pages.page))) return rc;
        const uint64_t qd = (uint64_t)p->config.q_heads * p->config.width;
        if ((rc = check_rows(p->q, p->q_stride, qd, "q"))) return rc;
        if ((rc = check_rows(p->out, p->out_stride, qd, "out"))) return rc;
        if (p->q == p->out) return fail(AF_ERR_INVALID, "out must not overlap q");
        if ((rc = check_workspace(p->workspace, need, stream))) return rc;
        PagedAttn a{};
        a.q = p->q;
        a.out = p->out;
        a.q_stride = p->q_stride;
        a.out_stride = p->out_stride;
        a.k_pages = (const uint8_t*)p->pages.k;
        a.v_pages = (const uint8_t*)p->pages.v;
        a.kv_heads = p->config.kv_heads;
        a.group = p->config.q_heads / p->config.kv_heads;
        a.window = p->config.window;
        a.sinks = p->sinks;
        a.scale = p->config.scale;
        a.b = batch_view(p->batch, p->pages);
        a.tickets = (uint32_t*)p->workspace->p;
        a.part = (float*)((char*)p->workspace->p + kTicketBytes);
        const AttnPlan plan = attn_plan(shape_of(*p));
        a.ticket_stride = ticket_stride((uint64_t)plan.slots * a.kv_heads);
        const hipError_t e = launch_paged_attention(a, p->config.width, p->pages.type == AF_KV_Q4, plan, (hipStream_t)stream);
        return e == hipSuccess ? AF_OK : fail(e, "paged attention launch");
    });
}

int af_logits_select_workspace(const af_logits_args* p, size_t* bytes) {
    return guarded([&]() -> int {
        if (!p || !bytes) return fail(AF_ERR_INVALID, "null argument");
        if (p->rows == 0 || p->rows > AF_MAX_LOGIT_ROWS || p->vocabulary == 0 || p->vocabulary > 0x1000000u)
            return fail(AF_ERR_INVALID, "invalid number of rows or tokens of the vocabulary");
        if ((uint64_t)p->rows * p->vocabulary > 1ull << 34) return fail(AF_ERR_INVALID, "rows times vocabulary above 2^34");
        *bytes = kTicketBytes + (size_t)p->rows * ((p->vocabulary + kLogitsSlice - 1) / kLogitsSlice) * 16;
        return AF_OK;
    });
}

int af_logits_select(const af_logits_args* p, void* stream) {
    return guarded([&]() -> int {
        size_t need = 0;
        int rc = af_logits_select_workspace(p, &need);
        if (rc) return rc;
        if (!p->logits || !p->result) return fail(AF_ERR_INVALID, "null logits or result");
        if (p->stride < p->vocabulary || (p->out && p->out_stride < p->vocabulary))
            return fail(AF_ERR_INVALID, "rows of logits overlap: the stride is less than the vocabulary");
        if (p->out == p->logits && p->out_stride != p->stride)
            return fail(AF_ERR_INVALID, "out in place of the logits must have their stride");
        if (p->history && (!p->history_len || p->history_stride == 0 || p->history_stride > AF_MAX_HISTORY))
            return fail(AF_ERR_INVALID, "a history needs its lengths and a stride of 1 to 65535 ids");
        if (p->bias_ids && (!p->bias_values || !p->bias_len || p->bias_stride == 0 || p->bias_stride > AF_MAX_HISTORY))
            return fail(AF_ERR_INVALID, "biases need their values, lengths and a stride of 1 to 65535 ids");
        if (p->mask && p->mask_stride < (p->vocabulary + 31) / 32)
            return fail(AF_ERR_INVALID, "a mask row must hold a bit for every token");
        if ((rc = check_workspace(p->workspace, need, stream))) return rc;
        LogitsSelect a{};
        a.logits = p->logits;
        a.out = p->out;
        a.stride = p->stride;
        a.out_stride = p->out_stride;
        a.rows = p->rows;
        a.vocabulary = p->vocabulary;
        a.penalties = p->penalties;
        a.history = p->history;
        a.history_len = p->history_len;
        a.history_stride = p->history_stride;
        a.bias_ids = p->bias_ids;
        a.bias_values = p->bias_values;
        a.bias_len = p->bias_len;
        a.bias_stride = p->bias_stride;
        a.mask = p->mask;
        a.mask_stride = p->mask_stride;
        a.result = p->result;
        a.tickets = (uint32_t*)p->workspace->p;
        a.part = (uint4*)((char*)p->workspace->p + kTicketBytes);
        a.ticket_stride = ticket_stride(p->rows);
        a.slices = (p->vocabulary + kLogitsSlice - 1) / kLogitsSlice;
        const hipError_t e = launch_logits_select(a, (hipStream_t)stream);
        return e == hipSuccess ? AF_OK : fail(e, "logits launch");
    });
}

}  // extern "C"
