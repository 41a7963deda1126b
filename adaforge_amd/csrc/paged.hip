// The paged KV cache of several sequences: appending to it (norms, RoPE, fp16 or 4-bit blocks), reading it back, and
// attention over it.
#include "device.h"
#include "paged.h"

namespace af {

namespace {

// ---- where a batch's rows stand ------------------------------------------------------------------

// The sequence whose rows hold row `token` (wave-uniform; the last s with starts[s] <= token), searched 64 ways at a
// time: one round of loads for up to 64 sequences.
__device__ __forceinline__ uint32_t sequence_of(const PagedBatch& b, uint32_t token) {
    uint32_t lo = 0, n = b.sequences;
    const uint32_t lane = threadIdx.x & 63;
    while (n > 1) {
        const uint32_t step = (n + 63) / 64, i = lane * step;
        const bool at = i < n && b.starts[lo + i] <= token;
        const uint32_t k = __popcll(__ballot(at));
        const uint32_t skip = k ? (k - 1) * step : 0;
        lo += skip;
        n = min(step, n - skip);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

struct Place {
    uint32_t seq;
    int32_t pos;
    bool row;  // the row belongs to a sequence
};

__device__ __forceinline__ Place place_of(const PagedBatch& b, uint32_t token) {
    Place p;
    p.seq = sequence_of(b, token);
    const Span s = span_of(b.starts[p.seq], b.starts[p.seq + 1], b.lengths[p.seq], b);
    p.row = token >= s.first && token - s.first < s.count;
    p.pos = s.pos0 + (int32_t)(token - s.first);
    return p;
}

// The page of position pos (0 .. table_stride * page - 1), or one past the last.
__device__ __forceinline__ uint32_t page_of(const PagedBatch& b, uint32_t seq, int32_t pos) {
    const uint32_t e = (uint32_t)pos >> b.page_shift;
    if (pos < 0 || e >= b.table_stride) return b.pages;
    return min(b.table[(size_t)seq * b.table_stride + e], b.pages);
}

// ---- 4-bit blocks ----------------------------------------------------------------------------------

typedef _Float16 h2 __attribute__((ext_vector_type(2)));

// The fp16 values of a word's eight codes under scale d: pairs (2 i, 2 i + 1) at bits 4 i and 16 + 4 i.  A code n in
// the low bits of 0x6400 is the fp16 number 1024 + n, so n - 8 is one exact subtraction, and d (n - 8) one rounding.
__device__ __forceinline__ void unpack4(uint32_t w, _Float16 d, h2 (&o)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t b = (w >> (4 * i) & 0x000F000Fu) | 0x64006400u;
        const h2 n = __builtin_bit_cast(h2, b) - h2{(_Float16)1032.0f, (_Float16)1032.0f};
        o[i] = n * h2{d, d};
    }
}

// ---- append -----------------------------------------------------------------------------------------
//
// A wave takes one head's row of a token: its sum of squares in 64 bits, then each pair's rotation, one rounding to
// f32, and for K and V the cache's type.  An angle is position times turns mod 2^64 as a fraction of a turn: a
// product that wraps keeps exactly the part that sine and cosine see, so far positions lose nothing and no general
// argument reduction is needed.

template <int W, bool Q4>
__global__ __launch_bounds__(256) void kv_append_kernel(KvAppend a, uint32_t groups, uint32_t tasks) {
    constexpr int P = W / 128 ? W / 128 : 1, HALF = W / 2;  // pairs per lane
    __shared__ __align__(16) float rows[4][W];
    const uint32_t lane = threadIdx.x & 63, wave = wave_id(), heads = a.q_heads + 2 * a.kv_heads;
    for (uint32_t task = blockIdx.x; task < tasks; task += gridDim.x) {
        const uint32_t token = task / groups, r = task % groups * 4 + wave;
        if (r >= heads) continue;
        const Place at = place_of(a.b, token);
        if (!at.row) continue;
        const bool is_q = r < a.q_heads, is_v = r >= a.q_heads + a.kv_heads;
        const uint32_t head = is_q ? r : is_v ? r - a.q_heads - a.kv_heads : r - a.q_heads;
        const float* src = is_q ? a.q + (size_t)token * a.q_stride
                                : is_v ? a.v + (size_t)token * a.v_stride : a.k + (size_t)token * a.k_stride;
        src += (size_t)head * W;
        const float* w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
        const float eps = is_q ? a.q_eps : is_v ? a.v_eps : a.k_eps;
        const bool norm = is_v ? a.v_norm != 0 : w != nullptr, on = (int)lane * P < HALF;
        float x[2][P];
        double ss = 0.0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < P; ++i) {
                x[h][i] = on ? src[h * HALF + lane * P + i] : 0.0f;
                ss = __fma_rn((double)x[h][i], (double)x[h][i], ss);
            }
        const double rn = norm ? inv_rms(wave_sum(ss), W, eps) : 1.0;
        const uint64_t* turns = is_v ? nullptr : a.turns;
        float y[2][P];
        if (on) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int c = lane * P + i;
                double u = (double)x[0][i], v = (double)x[1][i];
                if (norm) {
                    u *= rn;
                    v *= rn;
                }
                if (w) {
                    u *= (double)w[c];
                    v *= (double)w[HALF + c];
                }
                if (turns) {
                    const int64_t t = (int64_t)((uint64_t)(int64_t)at.pos * turns[c]);
                    double sn, cs;
                    sincospi((double)t * 0x1p-63, &sn, &cs);
                    const double u1 = u * cs - v * sn;
                    v = u * sn + v * cs;
                    u = u1;
                }
                y[0][i] = (float)u;
                y[1][i] = (float)v;
            }
        }
        if (is_q) {
            float* dst = a.q_out + (size_t)token * a.q_out_stride + (size_t)head * W;
            if (on)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < P; ++i) dst[h * HALF + lane * P + i] = y[h][i];
            continue;
        }
        const uint32_t page = page_of(a.b, at.seq, at.pos);
        if (page >= a.b.pages) continue;
        const uint32_t tokens = 1u << a.b.page_shift, slot = (uint32_t)at.pos & (tokens - 1);
        uint8_t* dst = (is_v ? a.v_pages : a.k_pages) +
                       ((size_t)page * a.kv_heads + head) * page_part_bytes(Q4, tokens, W);
        if constexpr (!Q4) {
            uint16_t* d16 = reinterpret_cast<uint16_t*>(dst) + (size_t)slot * W;
            if (on)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < P; ++i) d16[h * HALF + lane * P + i] = f2h(y[h][i]);
        } else {
            // through the wave's own LDS row: lane c then holds values 8 c .. 8 c + 7, four lanes a block
            if (on)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < P; ++i) rows[wave][h * HALF + lane * P + i] = y[h][i];
            __builtin_amdgcn_wave_barrier();
            if (lane < W / 8) {
                float e[8], high = -INFINITY, low = INFINITY;
                bool bad = false;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    e[i] = rows[wave][8 * lane + i];
                    high = fmaxf(high, e[i]);
                    low = fminf(low, e[i]);
                    bad |= !(fabsf(e[i]) < INFINITY);
                }
#pragma unroll
                for (int s = 1; s < 4; s <<= 1) {
                    high = fmaxf(high, __shfl_xor(high, s));
                    low = fminf(low, __shfl_xor(low, s));
                    bad |= __shfl_xor((int)bad, s) != 0;
                }
                uint16_t d = f2h((high >= -low ? high : low) / -8.0f);
                if (bad || (d & 0x7C00) == 0x7C00) d = 0x7E00;  // not finite: the block stands for NaNs
                const double scale = (double)h2f(d);
                uint32_t word = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const double n = scale == 0.0 || (d & 0x7C00) == 0x7C00
                                         ? 8.0
                                         : fmin(fmax(rint((double)e[i] / scale) + 8.0, 0.0), 15.0);
                    word |= (uint32_t)n << (4 * (i / 2) + 16 * (i & 1));
                }
                reinterpret_cast<uint32_t*>(dst)[(size_t)slot * (W / 8) + lane] = word;
                if (lane % 4 == 0)
                    reinterpret_cast<uint16_t*>(dst + (size_t)tokens * (W / 2))[slot * (W / 32) + lane / 4] = d;
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// Eight values 8 c .. 8 c + 7 of a cached row.
template <int W, bool Q4>
__device__ __forceinline__ v4u row_octet(const uint8_t* part, uint32_t tokens, uint32_t slot, uint32_t c) {
    if constexpr (!Q4) {
        return *reinterpret_cast<const v4u*>(part + ((size_t)slot * W + 8 * c) * 2);
    } else {
        const uint32_t w = reinterpret_cast<const uint32_t*>(part)[slot * (W / 8) + c];
        const uint16_t d = reinterpret_cast<const uint16_t*>(part + (size_t)tokens * (W / 2))[slot * (W / 32) + c / 4];
        h2 o[4];
        unpack4(w, __builtin_bit_cast(_Float16, d), o);
        return v4u{__builtin_bit_cast(uint32_t, o[0]), __builtin_bit_cast(uint32_t, o[1]),
                   __builtin_bit_cast(uint32_t, o[2]), __builtin_bit_cast(uint32_t, o[3])};
    }
}

template <int W, bool Q4>
__global__ __launch_bounds__(256) void kv_read_kernel(const uint8_t* k_pages, const uint8_t* v_pages, PagedBatch b,
                                                      uint32_t kv_heads, uint16_t* k, uint16_t* v) {
    for (uint32_t token = blockIdx.x; token < b.tokens; token += gridDim.x) {
        const Place at = place_of(b, token);
        if (!at.row) continue;
        const uint32_t page = page_of(b, at.seq, at.pos), tokens = 1u << b.page_shift, slot = (uint32_t)at.pos & (tokens - 1);
        const uint32_t n = kv_heads * (W / 8);
        for (uint32_t i = threadIdx.x; i < 2 * n; i += 256) {
            const uint32_t j = i < n ? i : i - n, head = j / (W / 8), c = j % (W / 8);
            v4u o = {0u, 0u, 0u, 0u};
            if (page < b.pages)
                o = row_octet<W, Q4>((i < n ? k_pages : v_pages) + ((size_t)page * kv_heads + head) * page_part_bytes(Q4, tokens, W),
                                     tokens, slot, c);
            *reinterpret_cast<v4u*>((i < n ? k : v) + ((size_t)token * kv_heads + head) * W + 8 * c) = o;
        }
    }
}

// ---- attention, key by key ----------------------------------------------------------------------------

// Softmax attention of one query by one wave, key by key in fp32 over key tiles [t0, t1) of T keys: values are read
// only where the query sees them.  Lane: channels E lane .. E lane + E - 1 (E = W / 64).
template <int W, bool Q4, uint32_t T>
__device__ void plain_row(const PagedAttn& a, const Tiles& tiles, uint32_t t0, uint32_t t1, uint32_t seq, uint32_t h,
                          int32_t pos, uint32_t end, const float (&q)[W / 64], float (&acc)[W / 64], float& m, float& l) {
    constexpr int E = W / 64;
    const uint32_t lane = threadIdx.x & 63, tokens = 1u << a.b.page_shift;
    const uint32_t bytes = page_part_bytes(Q4, tokens, W);
    auto row = [&](const uint8_t* part, uint32_t slot, float (&o)[E]) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t c = E * lane + e;
            if constexpr (!Q4) {
                o[e] = h2f(reinterpret_cast<const uint16_t*>(part)[(size_t)slot * W + c]);
            } else {
                const uint32_t w = reinterpret_cast<const uint32_t*>(part)[slot * (W / 8) + c / 8];
                const int n = (int)(w >> (c % 8 / 2 * 4 + c % 2 * 16) & 15) - 8;
                const float d = h2f(reinterpret_cast<const uint16_t*>(part + (size_t)tokens * (W / 2))[slot * (W / 32) + c / 32]);
                o[e] = h2f(f2h(d * (float)n));
            }
        }
    };
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    m = -INFINITY;
    l = 0.0f;
    for (uint32_t t = t0; t < t1; ++t) {
        const uint32_t j0 = tile_at(tiles, t) * T;
        for (uint32_t j = j0; j < min(j0 + T, end); ++j) {
            if (!sees(pos, (int32_t)j, a.window, a.sinks)) continue;
            const uint32_t page = page_of(a.b, seq, (int32_t)j);
            if (page >= a.b.pages) continue;
            const uint32_t slot = j & (tokens - 1);
            const size_t off = ((size_t)page * a.kv_heads + h) * bytes;
            float v[E], d = 0.0f;
            row(a.k_pages + off, slot, v);
#pragma unroll
            for (int e = 0; e < E; ++e) d = fmaf(q[e], v[e], d);
            const float s = wave_sum(d) * a.scale, mn = fmaxf(m, s);
            const float p = s == -INFINITY ? 0.0f : expf(s - mn), al = mn == -INFINITY ? 1.0f : expf(m - mn);
            l = fmaf(l, al, p);
            row(a.v_pages + off, slot, v);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = p > 0.0f || p != p ? fmaf(p, v[e], acc[e] * al) : acc[e] * al;
            m = mn;
            if (l != l) {  // every output is a NaN
                m = 0.0f;
                return;
            }
        }
    }
}

template <int W, bool Q4>
__global__ __launch_bounds__(64) void paged_attention_plain_kernel(PagedAttn a, uint32_t q_heads) {
    constexpr int E = W / 64;
    const uint32_t token = blockIdx.x / q_heads, qh = blockIdx.x % q_heads, lane = threadIdx.x;
    const uint32_t seq = sequence_of(a.b, token);
    const Span s = span_of(a.b.starts[seq], a.b.starts[seq + 1], a.b.lengths[seq], a.b);
    if (token < s.first || token - s.first >= s.count) return;
    const int32_t pos = s.pos0 + (int32_t)(token - s.first);
    const Tiles t = tiles_of<32>(pos, pos, s.end, a.window, a.sinks);
    float q[E], acc[E], m, l;
    for (int e = 0; e < E; ++e) q[e] = a.q[(size_t)token * a.q_stride + (size_t)qh * W + E * lane + e];
    plain_row<W, Q4, 32>(a, t, 0, t.count, seq, qh / a.group, pos, s.end, q, acc, m, l);
    float* o = a.out + (size_t)token * a.out_stride + (size_t)qh * W + E * lane;
    for (int e = 0; e < E; ++e) o[e] = l == 0.0f ? 0.0f : acc[e] / l;
}

}  // namespace

// ---- launches ----------------------------------------------------------------------------------------

// Calls f(width constant, 4-bit constant) for a supported width.
template <typename F>
static hipError_t by_layout(uint32_t width, bool q4, F f) {
    auto w = [&](auto c) { return q4 ? f(c, std::true_type{}) : f(c, std::false_type{}); };
    switch (width) {
        case 64: return w(std::integral_constant<int, 64>{});
        case 128: return w(std::integral_constant<int, 128>{});
        case 256: return w(std::integral_constant<int, 256>{});
        case 512: return w(std::integral_constant<int, 512>{});
    }
    return hipErrorInvalidValue;
}

hipError_t launch_kv_append(const KvAppend& a, uint32_t width, bool q4, hipStream_t s) {
    const uint32_t groups = (a.q_heads + 2 * a.kv_heads + 3) / 4, tasks = a.b.tokens * groups;
    return by_layout(width, q4, [&](auto w, auto t) {
        hipLaunchKernelGGL((kv_append_kernel<decltype(w)::value, decltype(t)::value>), dim3(min(tasks, 1u << 20)), dim3(256), 0,
                           s, a, groups, tasks);
        return hipGetLastError();
    });
}

hipError_t launch_kv_read(const uint8_t* k_pages, const uint8_t* v_pages, const PagedBatch& b, uint32_t kv_heads,
                          uint32_t width, bool q4, uint16_t* k, uint16_t* v, hipStream_t s) {
    return by_layout(width, q4, [&](auto w, auto t) {
        hipLaunchKernelGGL((kv_read_kernel<decltype(w)::value, decltype(t)::value>), dim3(b.tokens), dim3(256), 0, s, k_pages,
                           v_pages, b, kv_heads, k, v);
        return hipGetLastError();
    });
}

hipError_t launch_paged_attention(const PagedAttn& a, uint32_t width, bool q4, hipStream_t s) {
    const uint32_t q_heads = a.kv_heads * a.group;
    return by_layout(width, q4, [&](auto w, auto t) {
        hipLaunchKernelGGL((paged_attention_plain_kernel<decltype(w)::value, decltype(t)::value>), dim3(a.b.tokens * q_heads),
                           dim3(64), 0, s, a, q_heads);
        return hipGetLastError();
    });
}

}  // namespace af
