// The paged KV cache of several sequences: appending to it (norms, RoPE, fp16 or 4-bit blocks), reading it back, and
// attention over it.
#include "device.h"
#include "paged.h"

namespace af {

namespace {

// ---- where a batch's rows stand ------------------------------------------------------------------

// The last sequence s with before(s) true (wave-uniform; 0 if there is none), for before that holds up to some s:
// searched 64 ways at a time, one round of loads for up to 64 sequences.
template <typename F>
__device__ __forceinline__ uint32_t last_sequence(uint32_t sequences, F before) {
    uint32_t lo = 0, n = sequences;
    const uint32_t lane = threadIdx.x & 63;
    while (n > 1) {
        const uint32_t step = (n + 63) / 64, i = lane * step;
        const bool at = i < n && before(lo + i);
        const uint32_t k = __popcll(__ballot(at));
        const uint32_t skip = k ? (k - 1) * step : 0;
        lo += skip;
        n = min(step, n - skip);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// The last sequence with before(start, s) true, and its span: one round of loads for up to 64 sequences.  meanwhile()
// is called once the first loads are on their way.
template <typename F, typename G>
__device__ __forceinline__ uint32_t find_span(const PagedBatch& b, F before, Span& s, G meanwhile) {
    if (b.sequences <= 64) {
        const uint32_t i = min(threadIdx.x & 63, b.sequences - 1);
        const uint32_t start = *gp(b.starts + i), stop = *gp(b.starts + i + 1), length = *gp(b.lengths + i);
        __builtin_amdgcn_sched_barrier(0);
        meanwhile();
        const uint64_t at = __ballot((threadIdx.x & 63) < b.sequences && before(start, i));
        const uint32_t seq = __builtin_amdgcn_readfirstlane(max(1, __popcll(at)) - 1);
        s = span_of(__builtin_amdgcn_readlane(start, seq), __builtin_amdgcn_readlane(stop, seq), __builtin_amdgcn_readlane(length, seq), b);
        return seq;
    }
    meanwhile();
    const uint32_t seq = last_sequence(b.sequences, [&](uint32_t k) { return before(b.starts[k], k); });
    s = span_of(b.starts[seq], b.starts[seq + 1], b.lengths[seq], b);
    return seq;
}

struct Place {
    uint32_t seq;
    int32_t pos;
    bool row;  // the row belongs to a sequence
};

template <typename G>
__device__ __forceinline__ Place place_of(const PagedBatch& b, uint32_t token, G meanwhile) {
    Place p;
    Span s;
    p.seq = find_span(b, [&](uint32_t start, uint32_t) { return start <= token; }, s, meanwhile);
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
// the low bits of 0x6400 is the fp16 number 1024 + n, four bits higher 1024 + 16 n, so n - 8 is one exact operation,
// and d (n - 8) one rounding.
__device__ __forceinline__ void unpack4(uint32_t w, _Float16 d, h2 (&o)[4]) {
    // (in registers that the compiler does not know, mask and magic make one instruction; as constants two)
    uint32_t even = 0x000F000Fu, odd = 0x00F000F0u, magic = 0x64006400u;
    asm("" : "+s"(even), "+s"(odd), "+v"(magic));
    auto code = [&](uint32_t v, uint32_t mask) { return __builtin_bit_cast(h2, (v & mask) | magic); };
    const h2 low = {(_Float16)-1032.0f, (_Float16)-1032.0f}, high = {(_Float16)-72.0f, (_Float16)-72.0f};
    const h2 part = {(_Float16)0.0625f, (_Float16)0.0625f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t v = w >> (8 * i);
        o[2 * i] = (code(v, even) + low) * h2{d, d};
        o[2 * i + 1] = __builtin_elementwise_fma(code(v, odd), part, high) * h2{d, d};
    }
}

// ---- append -----------------------------------------------------------------------------------------
//
// A wave takes N heads' rows of a token: their sums of squares in 64 bits, then each pair's rotation, one rounding to
// f32, and for K and V the cache's type.  An angle is position times turns mod 2^64 as a fraction of a turn: a
// product that wraps keeps exactly the part that sine and cosine see, so far positions lose nothing and no general
// argument reduction is needed.  Its rows are on their way while the token's place is looked up.  N = 4 shares the sines
// among four rows and keeps four times the bytes in flight; N = 1 spreads a decode step over the chip.  Bound by 8 bytes
// per value of q, 4 and the cache's per value of k and v: four prompts (1,820 rows of 16 + 16 heads, 105 MB) 28.5 us =
// 3.7 TB/s, N = 1 45 us; by latency where there are few: one token 3.4 us, 64 tokens to 4 bits 6.3, N = 4 13.

template <int W, bool Q4, int N>
__global__ __launch_bounds__(256) void kv_append_kernel(KvAppend a, uint32_t groups, uint32_t tasks) {
    constexpr int P = W / 128 ? W / 128 : 1, HALF = W / 2;  // pairs per lane
    __shared__ __align__(16) float rows[Q4 ? 4 : 1][Q4 ? W : 4];
    const uint32_t lane = threadIdx.x & 63, wave = wave_id(), heads = a.q_heads + 2 * a.kv_heads;
    const bool on = (int)lane * P < HALF;
    for (uint32_t task = blockIdx.x; task < tasks; task += gridDim.x) {
        const uint32_t token = task / groups, r0 = (task % groups * 4 + wave) * N;
        if (r0 >= heads) continue;
        float x[N][2][P];
        uint64_t turn_of[P];
        const bool turned = a.turns && r0 < a.q_heads + a.kv_heads;
        const Place at = place_of(a.b, token, [&] {
            if (turned && on)
#pragma unroll
                for (int i = 0; i < P; ++i) turn_of[i] = a.turns[lane * P + i];
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const uint32_t r = min(r0 + k, heads - 1);
                const float* src = r < a.q_heads                  ? a.q + (size_t)token * a.q_stride + (size_t)r * W
                                   : r >= a.q_heads + a.kv_heads ? a.v + (size_t)token * a.v_stride + (size_t)(r - a.q_heads - a.kv_heads) * W
                                                                 : a.k + (size_t)token * a.k_stride + (size_t)(r - a.q_heads) * W;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < P; ++i) x[k][h][i] = on ? src[h * HALF + lane * P + i] : 0.0f;
            }
        });
        if (!at.row) continue;
        const uint32_t page = page_of(a.b, at.seq, at.pos), tokens = 1u << a.b.page_shift, slot = (uint32_t)at.pos & (tokens - 1);
        double sn[P], cs[P];
        if (turned && on)
#pragma unroll
            for (int i = 0; i < P; ++i)
                sincospi((double)(int64_t)((uint64_t)(int64_t)at.pos * turn_of[i]) * 0x1p-63, &sn[i], &cs[i]);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const uint32_t r = r0 + k;
            if (r >= heads) break;
            const bool is_q = r < a.q_heads, is_v = r >= a.q_heads + a.kv_heads;
            const uint32_t head = is_q ? r : is_v ? r - a.q_heads - a.kv_heads : r - a.q_heads;
            const float* w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
            const bool norm = is_v ? a.v_norm != 0 : w != nullptr, turn = turned && !is_v;
            float y[2][P];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < P; ++i) y[h][i] = x[k][h][i];
            if (norm || turn) {
                double rn = 1.0;
                if (norm) {
                    double ss = 0.0;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < P; ++i) ss = __fma_rn((double)x[k][h][i], (double)x[k][h][i], ss);
                    const float eps = is_q ? a.q_eps : is_v ? a.v_eps : a.k_eps;
                    ss = wave_sum(ss);
                    rn = ss < 1e300 ? inv_rms_fast(ss, W, eps) : inv_rms(ss, W, eps);  // (an infinite row: 0, as divided)
                }
                if (on)
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        const int c = lane * P + i;
                        double u = (double)x[k][0][i], v = (double)x[k][1][i];
                        if (norm) {
                            u *= rn;
                            v *= rn;
                        }
                        if (w) {
                            u *= (double)w[c];
                            v *= (double)w[HALF + c];
                        }
                        if (turn) {
                            const double u1 = u * cs[i] - v * sn[i];
                            v = u * sn[i] + v * cs[i];
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
            if (page >= a.b.pages) continue;
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
                    high = fmaxf(high, dpp<kDppXor1>(high));
                    high = fmaxf(high, dpp<kDppXor2>(high));
                    low = fminf(low, dpp<kDppXor1>(low));
                    low = fminf(low, dpp<kDppXor2>(low));
                    float odd = bad ? 1.0f : 0.0f;
                    odd = fmaxf(odd, dpp<kDppXor1>(odd));
                    odd = fmaxf(odd, dpp<kDppXor2>(odd));
                    uint16_t d = f2h((high >= -low ? high : low) / -8.0f);
                    if (odd != 0.0f || (d & 0x7C00) == 0x7C00) d = 0x7E00;  // not finite: the block stands for NaNs
                    // rint(e / d), exactly: a quotient good to 2^-22 is rounded to some n, whose remainder e - n d is exact
                    // (n d has 15 bits) and says whether the nearest is n or a neighbour (ties to even).  A scale of 0: all 8.
                    const bool plain = d != 0x7E00 && (d & 0x7FFF) != 0;
                    const float scale = h2f(d), inverse = plain ? 1.0f / scale : 0.0f, half = 0.5f * fabsf(scale);
                    uint32_t word = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float n = fminf(fmaxf(rintf(e[i] * inverse), -16.0f), 16.0f);
                        const float r = fmaf(-n, scale, e[i]), far = fabsf(r);
                        if (far > half || (far == half && ((int)n & 1))) n += (r < 0.0f) == (scale < 0.0f) ? 1.0f : -1.0f;
                        const int c = plain ? min(max((int)n + 8, 0), 15) : 8;
                        word |= (uint32_t)c << (4 * (i / 2) + 16 * (i & 1));
                    }
                    reinterpret_cast<uint32_t*>(dst)[(size_t)slot * (W / 8) + lane] = word;
                    if (lane % 4 == 0)
                        reinterpret_cast<uint16_t*>(dst + (size_t)tokens * (W / 2))[slot * (W / 32) + lane / 4] = d;
                }
                __builtin_amdgcn_wave_barrier();
            }
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
        const Place at = place_of(b, token, [] {});
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

constexpr float kLog2e = 1.44269504088896340736f, kLog2eLow = 1.92596299112661746887e-8f;  // log2(e), and what its float lacks

// ---- attention, key by key ----------------------------------------------------------------------------

// Softmax attention of one query by one wave, key by key in fp32 over key tiles t0, t0 + step, .. below t1:
// values are read only where the query sees them.  What the products below fall back to where a sum of theirs is
// not finite: there an infinite cached value meets halves of a pair that are zero or of the other sign, also
// of keys that the row does not see; and where scores are so large that fp32 holds them to no less than parts of a unit (far_off).
// Lane: channels E lane .. E lane + E - 1 (E = W / 64).  The sums are left as the products hold theirs, times 2^-m for a whole m (the
// nearest to the maximum in base 2, whose remainder goes into them: maxima of 2^30, held to 128, would else join
// as equals).
template <int W, bool Q4>
__device__ __forceinline__ void plain_row(const PagedAttn& a, const Tiles& tiles, uint32_t t0, uint32_t t1, uint32_t step,
                                          uint32_t seq, uint32_t h, int32_t pos, uint32_t end, const float (&q)[W / 64],
                                          float (&acc)[W / 64], float& m, float& l) {
#pragma clang fp contract(off)  // (a score less the maximum: both rounded, or the largest key's weight is not 1)
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
#pragma unroll 1
    for (uint32_t t = t0; t < t1; t += step) {
        const uint32_t j0 = tile_at(tiles, t) * 32;
#pragma unroll 1
        for (uint32_t j = j0; j < min(j0 + 32, end); ++j) {
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
            // (the weights, which lanes have alike, by lanes: thousands of like terms in one sum would all round the same way)
            l = fmaf(l, al, lane == (j & 63) ? p : 0.0f);
            row(a.v_pages + off, slot, v);
#pragma unroll
            for (int e = 0; e < E; ++e) {  // (no infinity times a weight of 0)
                const float kept = al != 0.0f ? acc[e] * al : 0.0f;
                acc[e] = p > 0.0f || p != p ? fmaf(p, v[e], kept) : kept;
            }
            m = mn;
            if (p != p) {  // every output is a NaN
                m = 0.0f;
                l = p;
                return;
            }
        }
    }
    l = wave_sum(l);
    if (m > -INFINITY) {
        const float whole = rintf(m * kLog2e), rest = fmaf(m, kLog2e, -whole) + m * kLog2eLow;
        // (a remainder past 60: from 2^30 on, where unequal maxima are further apart than 2^60 in their weights anyway)
        const float f = __builtin_amdgcn_exp2f(fminf(fmaxf(rest, -60.0f), 60.0f));
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= f;
        l *= f;
        m = whole;
    }
}

// ---- attention of few rows: single tokens, and short drafts over few keys --------------------------------
//
// Rows are the (token, query head) pairs that share a KV head: row i of a sequence is token i / group, head i % group.
// A block takes 16 of them against a chunk of the sequence's key tiles, its four waves tile by tile in turn; the
// chunks of one row tile meet at a ticket, where the last block joins their partial sums (one pass over the
// data with a running maximum and sum).  Bound by reading K and V once: one token at 32,768 positions (8 heads of 256,
// fp16, 268 MB) 50.2 us = 5.3 TB/s, 32 of 1 to 8,192 positions 194 us = 5.5 TB/s; 4-bit rows by unpacking them (13
// instructions a word of eight) and by the waits between dependent steps: 64 windows of 1,024 41.8 us = 3.6 TB/s, eight
// 512-wide heads of up to 32,768 positions (a block a CU) 35 us and 7 the join; short contexts by the chain of the
// sequence's place, the page numbers, K, V, the ticket and the join: one token at 512 positions 10.4 us.
//
// Products are taken transposed on the fp16 matrix cores, S^T = K Q^T and O^T = V^T P^T (16 keys or channels by 16
// rows): a lane holds one row's column throughout (row lane % 16), so the softmax needs lane swaps only
// where its reference moves, and P is the second product's operand as it stands.  The order of the channels in the first sum and of the
// keys in the second is free: lane group g = lane / 16 takes the channels its own 16-byte loads bring, and keys
// 4 g .. 4 g + 3 of each half of a tile, so that K and V go from memory to operands in registers without LDS; V's
// pairs of keys are made by byte permutes.  A half of a tile lies in one page (pages hold at least 16 tokens), so its
// base address is scalar and every load adds a constant per lane.
//
// fp32 rows enter as fp16 pairs hi + lo: queries scaled by a power of two (pair_scale), weights by one that the exponent takes
// in (Softmax).

constexpr int kPartSC1 = 16;      // buffer access policy sc1: through to (or from) the memory side
constexpr int kWaitVm0 = 0x0F70;  // s_waitcnt vmcnt(0), expcnt and lgkmcnt unconstrained

// The first key that a query at position p sees, apart from the first tokens.
__device__ __forceinline__ int32_t first_seen(int32_t p, uint32_t window) {
    return window == 0 || window > 1u << 30 ? 0 : max(0, p + 1 - (int32_t)window);
}

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float lanes4_max(float v) {
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float w = fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
    const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(w), __float_as_uint(w), false, false);
    return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}

// Two floats to nearest fp16, and x less one of them (exact: one instruction takes the fp16 operand as it is).
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{a, b}, h2));
}
template <int HALF>
__device__ __forceinline__ float less_half(float x, uint32_t h) {
    float r;
    if constexpr (HALF == 0)
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    else
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    return r;
}

// The power of two that brings a query whose largest element is mx to 2^14 .. 2^15: a pair then has 22 bits of every element down to
// 2^-17 of the largest, and 2^-40 of that of smaller ones (one channel 1e5 times the others where the keys are zero: 4e-7
// of the output wrong, with the largest below 32 8e-5).  At most 2^126, so that it and its reciprocal are finite.
__device__ __forceinline__ float pair_scale(float mx) {
    return mx > 0.0f ? ldexpf(1.0f, min(14 - ilogbf(mx), 126)) : 1.0f;
}

// The step and lane group whose operand holds channels 8 o .. 8 o + 7 of a key's row.
template <int W, bool Q4>
__device__ __forceinline__ void operand_of(uint32_t o, uint32_t& step, uint32_t& g) {
    if constexpr (!Q4) {
        step = o / 4;
        g = o % 4;
    } else if constexpr (W >= 128) {  // a lane's 16-byte load of codes is one block of 32 channels: four steps
        step = o / 16 * 4 + o % 4;
        g = o / 4 % 4;
    } else {
        step = o % 2;
        g = o / 2;
    }
}

// Where 32 tiles' halves (16 keys, in one page) lie: lane l holds that of half l % 2 of tile first + l / 2 step, so that
// the table is read, and an offset computed, once in 32 tiles; a tile's base addresses are then lane reads.
template <int W, bool Q4>
struct HalfTable {
    uint32_t lo, hi;  // byte offset of the half's first row (of codes) in the pages
    uint32_t scales;  // 4 bits: from there to its first row of scales
    uint64_t ok;      // lanes whose half has a page (others: some page, nothing of which is seen)
    uint32_t first;

    __device__ __forceinline__ void fill(const PagedAttn& a, const Tiles& keys, uint32_t seq, uint32_t h, uint32_t t, uint32_t step,
                                         uint32_t end) {
        const uint32_t lane = threadIdx.x & 63, tokens = 1u << a.b.page_shift;
        const uint32_t j = tile_at(keys, min(t + lane / 2 * step, end - 1)) * 32 + lane % 2 * 16, e = j >> a.b.page_shift;
        const uint32_t page = e < a.b.table_stride ? a.b.table[(size_t)seq * a.b.table_stride + e] : a.b.pages;
        const uint32_t slot = j & (tokens - 1);
        const uint64_t off = ((uint64_t)(page < a.b.pages ? page : 0) * a.kv_heads + h) * page_part_bytes(Q4, tokens, W) +
                             slot * (Q4 ? W / 2 : W * 2);
        ok = __ballot(page < a.b.pages);
        lo = (uint32_t)off;
        hi = (uint32_t)(off >> 32);
        scales = tokens * (W / 2) + slot * (W / 16) - slot * (W / 2);
        first = t;
    }
    __device__ __forceinline__ uint64_t offset(uint32_t l) const {
        return (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, l) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, l);
    }
    __device__ __forceinline__ uint32_t scales_at(uint32_t l) const { return Q4 ? __builtin_amdgcn_readlane(scales, l) : 0; }
};

// A load of rows that no other block reads (NT: past the caches' keeping).  One token at 32,768 positions 57.6 -> 53.7 us,
// 16 sequences of 8,192 in 128-wide heads 101 -> 94; where row tiles share the rows 25.5 -> 28.2 us (three of them, 4,096
// positions), and 4-bit rows, whose lines two loads share, 56 -> 57, so neither is loaded so.
template <bool NT, typename T>
__device__ __forceinline__ T load_row(const __attribute__((address_space(1))) T* p) {
    if constexpr (NT)
        return __builtin_nontemporal_load(p);
    else
        return *p;
}

// Rows of K of one half tile (16 keys): a lane's loads, and its operand of a step.
template <int W, bool Q4, bool NT>
struct KHalf {
    v4u f[Q4 ? 1 : W / 32];
    v4u c[Q4 ? (W >= 128 ? W / 128 : 1) : 1];
    uint32_t d[Q4 ? (W >= 128 ? W / 128 : 1) : 1];  // (fp16 scales)

    // rows: of the half (4 bits: codes), scales: from there to its scales
    __device__ __forceinline__ void load(const uint8_t* rows, uint32_t scales, uint32_t lane) {
        const uint32_t m = lane & 15, g = lane >> 4;
        if constexpr (!Q4) {
            const auto* p = gp(rows) + (m * (W * 2) + g * 16);
#pragma unroll
            for (int s = 0; s < W / 32; ++s) f[s] = load_row<NT>((const __attribute__((address_space(1))) v4u*)(p + 64 * s));
        } else {
            const auto* sc = gp(rows + scales);
            const auto* p = gp(rows);
            if constexpr (W >= 128) {
#pragma unroll
                for (int i = 0; i < W / 128; ++i) {
                    c[i] = *(const __attribute__((address_space(1))) v4u*)(p + (m * (W / 2) + g * 16 + 64 * i));
                    d[i] = *(const __attribute__((address_space(1))) uint16_t*)(sc + (m * (W / 16) + g * 2 + 8 * i));
                }
            } else {
                const u2 w = *(const __attribute__((address_space(1))) u2*)(p + (m * (W / 2) + g * 8));
                c[0] = v4u{w.x, w.y, 0u, 0u};
                d[0] = *(const __attribute__((address_space(1))) uint16_t*)(sc + (m * (W / 16) + g / 2 * 2));
            }
        }
    }
    __device__ __forceinline__ h8 operand(int s) const {
        if constexpr (!Q4) {
            return __builtin_bit_cast(h8, f[s]);
        } else {
            h2 o[4];
            unpack4(c[s / 4][s % 4], __builtin_bit_cast(_Float16, (uint16_t)d[s / 4]), o);
            return h8{o[0].x, o[0].y, o[1].x, o[1].y, o[2].x, o[2].y, o[3].x, o[3].y};
        }
    }
};

// V of one half tile: a lane's four keys (4 g + j), channels 16 E (t / E) + E m + t % E of tile t in 0 .. W / 16 - 1.
template <int W, bool Q4, bool NT>
struct VHalf {
    static constexpr int E = Q4 ? W / 16 : (W / 16 < 8 ? W / 16 : 8);  // channels a load brings
    static constexpr int C = W / 16 / E, R = Q4 ? (W / 128 ? W / 128 : 1) : E / 2;
    uint32_t w[4][C][R];
    uint32_t d[Q4 ? 4 : 1];  // (fp16 scales)

    __device__ __forceinline__ void load(const uint8_t* rows, uint32_t scales, uint32_t lane) {
        const uint32_t m = lane & 15, g = lane >> 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (!Q4) {
                const auto* p = gp(rows) + (g * (W * 8) + m * (2 * E) + j * (W * 2));
#pragma unroll
                for (int c = 0; c < C; ++c)
                    if constexpr (E == 8) {
                        const v4u x = load_row<NT>((const __attribute__((address_space(1))) v4u*)(p + 256 * c));
                        w[j][c][0] = x.x, w[j][c][1] = x.y, w[j][c][2] = x.z, w[j][c][3] = x.w;
                    } else {
                        const u2 x = *(const __attribute__((address_space(1))) u2*)(p);
                        w[j][c][0] = x.x, w[j][c][1] = x.y;
                    }
            } else {
                const auto* p = gp(rows) + (g * (W * 2) + m * (W / 32) + j * (W / 2));
                if constexpr (W == 512) {
                    const v4u x = *(const __attribute__((address_space(1))) v4u*)(p);
                    w[j][0][0] = x.x, w[j][0][1] = x.y, w[j][0][2] = x.z, w[j][0][3] = x.w;
                } else if constexpr (W == 256) {
                    const u2 x = *(const __attribute__((address_space(1))) u2*)(p);
                    w[j][0][0] = x.x, w[j][0][1] = x.y;
                } else if constexpr (W == 128) {
                    w[j][0][0] = *(const __attribute__((address_space(1))) uint32_t*)(p);
                } else {  // four of a word's eight: pairs 0 and 1, or 2 and 3
                    const auto* q = gp(rows) + (g * (W * 2) + m / 2 * 4 + j * (W / 2));
                    w[j][0][0] = *(const __attribute__((address_space(1))) uint32_t*)(q) >> (m % 2 * 8);
                }
                d[j] = *(const __attribute__((address_space(1))) uint16_t*)(gp(rows + scales) + (g * (W / 4) + m * W / 512 * 2 + j * (W / 16)));
            }
        }
    }
    // The lane's key j stands for zeros.
    __device__ __forceinline__ void clear(int j) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int r = 0; r < R; ++r) w[j][c][r] = 0;
        if constexpr (Q4) d[j] = 0;
    }
    // Operands of tiles 8 o .. (one octet of the lane's channels): per channel the halves' keys j, as pairs.
    template <int N>
    __device__ __forceinline__ void octet(int o, uint32_t (&k)[N][2]) const {
        uint32_t x[4][N / 2];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (!Q4) {
#pragma unroll
                for (int r = 0; r < N / 2; ++r) x[j][r] = w[j][o][r];
            } else {
                h2 p[4];
                unpack4(w[j][0][o], __builtin_bit_cast(_Float16, (uint16_t)d[j]), p);
#pragma unroll
                for (int r = 0; r < N / 2; ++r) x[j][r] = __builtin_bit_cast(uint32_t, p[r]);
            }
        }
#pragma unroll
        for (int e = 0; e < N; ++e)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                k[e][i] = __builtin_amdgcn_perm(x[2 * i + 1][e / 2], x[2 * i][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
    }
};

// The column's running softmax (base 2): weights 2^(score - m), as fp16 pairs, which have 22 bits from 2^-3 up to 2^16.  So m, a whole
// number, follows the tiles: where a tile's largest weight would be above 2^kHigh or below 1, m moves and the sums are rescaled
// (exactly).  It moves to make that weight about 2^kSet, which later tiles seldom leave; or 2^kAlone where one lane's eight keys stand
// kApart above another's: a key that may have most of the weight for itself, beside which the others' bits matter if its value
// is small.  And it moves down again behind such a key: first tokens that draw nearly all of the weight and add nothing leave an
// output of the others' weights.  2,500 keys, the first with a share of 0.9995 and a value of zero: 5e-7 of the output wrong in
// one chunk, 4e-6 to 2e-4 against one maximum that only rises.  But m stays within 2^kBack of its highest, so that the sums do not
// overflow: weights that lose bits by that are below 2^-68 of the sum.
constexpr float kSet = 8.0f, kAlone = 14.0f, kApart = 8.0f, kHigh = 15.5f, kBack = 60.0f;
constexpr float kNone = -3.402823466e38f;  // m of a column that has seen nothing

struct Softmax {
    float m = kNone, top = kNone, l = 0.0f;  // top: the highest m; l: the sum over this lane's keys

    // Takes in the lane's scores of eight keys (times qs; -inf: not seen): scale(f) gets the factor of the sums so far
    // where it is not 1 (lanes of a column agree).
    template <typename F>
    __device__ __forceinline__ void follow(const f4 (&s)[2], float qs, F scale) {
        const float mine = qs * fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                                      fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        if (__ballot(!(fabsf(mine - m - 0.5f * kHigh) <= 0.5f * kHigh))) {
            const uint64_t low = __ballot(!(mine - m >= 0.0f)), lows = low & low >> 32;  // (a column is low where its four lanes are)
            if (!(__ballot(mine - m > kHigh) | (lows & lows >> 16 & 0xFFFF))) return;
            const float mx = lanes4_max(mine), over = mx - m;
            const bool alone = mx + lanes4_max(mine > -INFINITY ? -mine : -INFINITY) > kApart;
            const float to = over > kHigh || (over < 0.0f && mx > -INFINITY) ? fmaxf(rintf(mx - (alone ? kAlone : kSet)), top - kBack) : m;
            if (__ballot(to != m)) {
                const float al = __builtin_amdgcn_exp2f(m - to);
                m = to;
                top = fmaxf(top, to);
                if (__ballot(l != 0.0f)) {  // (not for a wave's first tile)
                    l *= al;
                    scale(al);
                }
            }
        }
    }

    // Their weights, as fp16 pairs, in eight slices: 0 .. 3 two weights each, 4 .. 7 a pair's halves.
    struct Weights {
        float p[8];
        uint32_t hi[4], lo[4];
        __device__ __forceinline__ h8 high() const { return __builtin_bit_cast(h8, v4u{hi[0], hi[1], hi[2], hi[3]}); }
        __device__ __forceinline__ h8 low() const { return __builtin_bit_cast(h8, v4u{lo[0], lo[1], lo[2], lo[3]}); }
    };
    __device__ __forceinline__ void slice(int k, const f4 (&s)[2], float qs, Weights& w) {
        if (k < 4) {
#pragma unroll
            for (int e = 0; e < 2; ++e) w.p[2 * k + e] = __builtin_amdgcn_exp2f(fmaf(s[k / 2][k % 2 * 2 + e], qs, -m));
        } else {
            k -= 4;
            w.hi[k] = pack_f16(w.p[2 * k], w.p[2 * k + 1]);
            w.lo[k] = pack_f16(less_half<0>(w.p[2 * k], w.hi[k]), less_half<1>(w.p[2 * k + 1], w.hi[k]));
            if (k == 3) l += ((w.p[0] + w.p[1]) + (w.p[2] + w.p[3])) + ((w.p[4] + w.p[5]) + (w.p[6] + w.p[7]));
        }
    }
    __device__ __forceinline__ void weights(const f4 (&s)[2], float qs, Weights& w) {
#pragma unroll
        for (int k = 0; k < 8; ++k) slice(k, s, qs, w);
    }

    // Whether m is so far from 0 that its distance from scores is rounded (by 2^-3 at 2^21) and weights may leave fp16's range: above
    // 2^16, or all of them below 2^-24 while l has them.
    __device__ __forceinline__ bool far_off() const { return m > kNone && fabsf(m) > 0x1p21f; }
};

// The chunks of a row tile of `tiles` key tiles: chunk tiles each, or more where they would be over `splits`.
__device__ __forceinline__ void chunks_of(uint32_t tiles, uint32_t chunk, uint32_t splits, uint32_t& len, uint32_t& parts) {
    len = max(chunk, (tiles + splits - 1) / splits);
    parts = max(1u, (tiles + len - 1) / len);
}

// Rows c0, c0 + 4 / S, .. of a row tile from its chunks' partial sums [parts][R][W + 4] (sums, maximum, sum of weights), S
// waves a row: the chunks' weights first, a chunk per lane, then their sums, eight loads of a lane in flight and
// in the order of the chunks.  parts: at most 128.
template <int W, int S>
__device__ __forceinline__ void join_parts(const PagedAttn& a, const float* part, uint32_t parts, uint32_t R,
                                           uint32_t c0, uint32_t nr, uint32_t row0, uint32_t first, uint32_t h) {
    constexpr uint32_t Q = W / 4 / S, L = Q < 64 ? Q : 64, G = 64 / L, K = Q / L;  // a wave's quads, lanes of a row, chunks side by side, quads of a lane
    constexpr uint32_t U = 8 / K;                                               // chunks of a lane in flight
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(part), 0, (int)(parts * R * (W + 4) * 4), 0x00020000);
    const uint32_t lane = threadIdx.x & 63, x0 = wave_id() % S * Q;
    for (uint32_t c = c0 + wave_id() / S; c < nr; c += 4 / S) {
        v4u v[U][K];
        auto load = [&](uint32_t q0) {
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
#pragma unroll
                for (uint32_t k = 0; k < K; ++k)
                    v[u][k] = __builtin_amdgcn_raw_buffer_load_b128(
                        rs, ((min(q0 + lane / L + u * G, parts - 1) * R + c) * (W + 4) + (x0 + lane % L + L * k) * 4) * 4, 0, kPartSC1);
        };
        u2 ml[2];
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i)
            ml[i] = __builtin_amdgcn_raw_buffer_load_b64(rs, ((min(lane + 64 * i, parts - 1) * R + c) * (W + 4) + W) * 4, 0, kPartSC1);
        load(0);
        float m[2], l[2];
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            m[i] = lane + 64 * i < parts ? __uint_as_float(ml[i].x) : -INFINITY;
            l[i] = lane + 64 * i < parts ? __uint_as_float(ml[i].y) : 0.0f;
        }
        const float M = wave_max(fmaxf(m[0], m[1]));
        float f[2];  // (a chunk that saw nothing has maximum -inf and sum 0)
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) f[i] = m[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[i] - M);
        const float sum = wave_sum(f[0] * l[0] + f[1] * l[1]);
        f4 o[K];
#pragma unroll
        for (uint32_t k = 0; k < K; ++k) o[k] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t q0 = 0;;) {
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                const uint32_t p = q0 + lane / L + u * G;
                const float f0 = __shfl(f[0], p & 63), f1 = __shfl(f[1], p & 63), w = p >= parts ? 0.0f : p < 64 ? f0 : f1;
#pragma unroll
                for (uint32_t k = 0; k < K; ++k)
                    if (w != 0.0f) o[k] += w * __builtin_bit_cast(f4, v[u][k]);  // (no infinity times a weight of 0)
            }
            if ((q0 += U * G) >= parts) break;
            load(q0);
        }
#pragma unroll
        for (uint32_t d = L; d < 64; d <<= 1)
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) o[0][e] += __shfl_xor(o[0][e], d);
        const uint32_t row = row0 + c;
        float* out = a.out + (size_t)(first + row / a.group) * a.out_stride + (size_t)(h * a.group + row % a.group) * W;
        if (lane < L)
#pragma unroll
            for (uint32_t k = 0; k < K; ++k)
                *reinterpret_cast<f4*>(out + (x0 + lane + L * k) * 4) = sum == 0.0f ? f4{0.0f, 0.0f, 0.0f, 0.0f} : o[k] / sum;
    }
}

// The chunks of a unit meet at its ticket: whether this block's, whose partial sums are stored, is the last one in.  Where starts
// fall, units of several sequences may be one, with different numbers of chunks: no block of such a launch draws, so that
// every ticket is zero for the next (the starts are on their way while the sums are stored).
__device__ __forceinline__ bool last_chunk(const PagedAttn& a, uint32_t unit, uint32_t parts) {
    __shared__ uint32_t last;
    bool falls = false;
    if (wave_id() == 0)
        for (uint32_t i = threadIdx.x; i < a.b.sequences; i += 64) falls |= *gp(a.b.starts + i + 1) < *gp(a.b.starts + i);
    const bool draws = !__any(falls);
    __builtin_amdgcn_s_waitcnt(kWaitVm0);
    __syncthreads();
    if (threadIdx.x == 0) last = 0;
    if (threadIdx.x == 0 && draws) {
        uint32_t* t = a.tickets + unit * a.ticket_stride;
        last = __hip_atomic_fetch_add(t, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
        if (last) __hip_atomic_store(t, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return last;
}

// Sums over the lanes up to this one: within rows of 16 by shifts, then a row's last lane to the next row, lane 31's to the
// upper half.
__device__ __forceinline__ uint32_t wave_prefix(uint32_t v) {
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);  // row_shr by 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);  // row_bcast:15
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);  // row_bcast:31
    return v;
}

// n / d for n below 2^23, d > 0, rounded down.
__device__ __forceinline__ uint32_t quotient(uint32_t n, uint32_t d) {
    uint32_t q = (uint32_t)((float)n * __builtin_amdgcn_rcpf((float)d));  // (off by at most one)
    const int32_t rest = (int32_t)(n - q * d);
    return rest < 0 ? q - 1 : (uint32_t)rest >= d ? q + 1 : q;
}

// A sequence's part of what Shares deals out: `parts` chunks of `chunk` key tiles for each of its row tiles, the first
// of them chunk `first` of a KV head's.
struct Share {
    uint32_t seq, start, chunk, parts, first;
    Span s;
};

// The sequence for whose lane find(start, span, its first chunk, the end of its chunks) is true, or false.
template <typename F>
__device__ __forceinline__ bool share(const PagedAttn& a, const Shares& sh, uint32_t R, Share& o, F find) {
    const uint32_t lane = threadIdx.x & 63, i = min(lane, a.b.sequences - 1);
    const uint32_t start = *gp(a.b.starts + i), stop = *gp(a.b.starts + i + 1), length = *gp(a.b.lengths + i);
    const Span s = span_of(start, stop, length, a.b);
    const uint32_t r = lane < a.b.sequences ? (s.count * a.group + R - 1) / R : 0;
    const uint32_t n = r ? tiles_of<32>(s.pos0, s.pos0 + (int32_t)s.count - 1, s.end, a.window, a.sinks).count : 0;
    const uint32_t row_tiles = __builtin_amdgcn_readlane(wave_prefix(r), 63), total = __builtin_amdgcn_readlane(wave_prefix(r * n), 63);
    if (row_tiles > sh.slots) return false;  // (starts that do not rise)
    uint32_t chunk, c, end;  // key tiles of the lane's chunks, chunks of a row tile, end of all of them
    auto deal = [&](uint32_t per_fill) {
        chunk = share_chunk(share_of(sh, total, per_fill), n);
        c = max(1u, quotient(n + chunk - 1, chunk));
        end = wave_prefix(r * c);
        return (uint32_t)__builtin_amdgcn_readlane(end, 63);
    };
    // (equal lengths share evenly; others leave each row tile a smaller last chunk, and fill the chip with fewer)
    if (deal(sh.per_fill) > sh.most) deal(sh.per_safe);
    const uint64_t mine = __ballot(find(start, s, end - r * c, end));
    if (!mine) return false;
    const uint32_t l = __builtin_ctzll(mine);
    auto at = [&](uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)x, l); };
    o.seq = l;
    o.start = at(start);
    o.s = span_of(o.start, at(stop), at(length), a.b);
    o.chunk = at(chunk);
    o.parts = at(c);
    o.first = at(end - r * c);
    return true;
}

// join_apart: the chunks are joined by paged_join_kernel afterwards, not by the last of them.
template <int W, bool Q4, bool NT>
__global__ __launch_bounds__(256, W == 512 ? 1 : 2) void paged_few_kernel(PagedAttn a, uint32_t units, uint32_t splits,
                                                                          uint32_t row_tiles, uint32_t chunk, bool join_apart,
                                                                          Shares shares) {
    constexpr int ST = W / 32, TV = W / 16, HALFROWS = 8;
    using V = VHalf<W, Q4, NT>;
    // At the end eight rows of each wave's sums lie in LDS.  512 wide, with four floats behind every 4 E of them and rows 16
    // floats past a multiple of 64, so that a write's lanes (8 rows, 4 places 4 E apart) take different banks: eight
    // sequences of up to 32,768 positions 45.5 -> 43.8 us; 256 wide the addresses cost registers (52 -> 54 us).
    constexpr int SKEW = 4 * V::E, ROW = W == 512 ? (W + W / V::E - 16 + 63) / 64 * 64 + 16 : W;
    auto skewed = [](uint32_t x) { return W == 512 ? x + x / SKEW * 4 : x; };
    __shared__ __align__(16) uint8_t lds[4 * HALFROWS * ROW * 4];  // (the queries' operands before: 64 W bytes)
    __shared__ float wm[4][16], wl[4][16];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = wave_id(), m = lane & 15, g = lane >> 4;
    uint32_t h, seq, tile0, split, start, part0 = 0;  // part0: of the row tile's chunks, in shares
    Span s;
    if (shares.chunks) {
        h = blockIdx.x % a.kv_heads;
        const uint32_t b = blockIdx.x / a.kv_heads;
        Share o;
        if (!share(a, shares, 16, o, [&](uint32_t, const Span&, uint32_t first, uint32_t end) { return b >= first && b < end; })) return;
        seq = o.seq;
        start = o.start;
        s = o.s;
        chunk = o.chunk;
        const uint32_t r = (s.count * a.group + 15) / 16;
        split = __builtin_amdgcn_readfirstlane(quotient(b - o.first, r));
        tile0 = b - o.first - split * r;  // (a chunk's row tiles one after another: its K and V come from memory once)
        part0 = h * shares.chunks + o.first + tile0 * o.parts;
    } else {
        split = blockIdx.x / units;
        const uint32_t unit = blockIdx.x % units;
        h = unit % a.kv_heads;
        seq = unit / a.kv_heads % a.b.sequences;
        tile0 = unit / a.kv_heads / a.b.sequences;
        start = a.b.starts[seq];
        s = span_of(start, a.b.starts[seq + 1], a.b.lengths[seq], a.b);
    }
    const uint32_t rows = s.count * a.group;

    // (one turn unless a sequence has more rows than the launch was told)
    for (uint32_t rt = tile0; rt * 16 < rows; rt += row_tiles) {
        const uint32_t nr = min(16u, rows - rt * 16);
        const int32_t plo = s.pos0 + (int32_t)(rt * 16 / a.group), phi = s.pos0 + (int32_t)((rt * 16 + nr - 1) / a.group);
        const Tiles keys = tiles_of<32>(plo, phi, s.end, a.window, a.sinks);
        // the chunk of this block: at most `splits` of them
        uint32_t len, parts;
        chunks_of(keys.count, chunk, splits, len, parts);
        if (split >= parts) continue;
        const uint32_t t0 = split * len + wave, t1 = min((split + 1) * len, keys.count);

        HalfTable<W, Q4> where;  // of this wave's tiles
        struct Stage {
            KHalf<W, Q4, NT> k[2];
            V v[2];
            bool ok[2];
        } here;
        auto load_k = [&](uint32_t t, Stage& g) {
            if (t >= where.first + 128) where.fill(a, keys, seq, h, t, 4, keys.count);
            const uint32_t l = (t - where.first) / 2;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                g.ok[i] = where.ok >> (l + i) & 1;
                g.k[i].load(a.k_pages + where.offset(l + i), where.scales_at(l + i), lane);
            }
        };
        auto load_v = [&](uint32_t t, Stage& g) {
            const uint32_t l = (t - where.first) / 2;
#pragma unroll
            for (int i = 0; i < 2; ++i) g.v[i].load(a.v_pages + where.offset(l + i), where.scales_at(l + i), lane);
        };
        if (t0 < t1) {
            where.fill(a, keys, seq, h, t0, 4, keys.count);
            load_k(t0, here);
            load_v(t0, here);
        }

        // the queries as scaled fp16 pairs in operand order: thread (row tid / 16, lane of 16) takes octets of channels
        __syncthreads();  // (the last turn's sums are read)
        float qs;         // of this lane's column: what a product has to be multiplied by
        int32_t pos;
        {
            const uint32_t r = tid >> 4, c = tid & 15, row = rt * 16 + r;
            constexpr int N = W >= 128 ? W / 128 : 1;
            const bool on = r < nr && c < W / 8;
            const float* src = a.q + (size_t)(s.first + row / a.group) * a.q_stride + (size_t)(h * a.group + row % a.group) * W;
            float x[N][8], mx = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const f4 u = on ? *reinterpret_cast<const f4*>(src + 8 * (c + 16 * i)) : f4{0.0f, 0.0f, 0.0f, 0.0f};
                const f4 w = on ? *reinterpret_cast<const f4*>(src + 8 * (c + 16 * i) + 4) : f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[i][e] = u[e];
                    x[i][4 + e] = w[e];
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[i][e]));
            }
            const float up = pair_scale(row_max(mx));
            if (c < W / 8)
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    h8 hi, lo;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float y = x[i][e] * up;
                        hi[e] = (_Float16)y;
                        lo[e] = (_Float16)(y - (float)hi[e]);
                    }
                    uint32_t step, og;
                    operand_of<W, Q4>(c + 16 * i, step, og);
                    *reinterpret_cast<h8*>(lds + ((step * 2 + 0) * 64 + og * 16 + r) * 16) = hi;
                    *reinterpret_cast<h8*>(lds + ((step * 2 + 1) * 64 + og * 16 + r) * 16) = lo;
                }
            if (c == 0) wm[0][r] = a.scale / up * kLog2e;
            __syncthreads();
            qs = wm[0][m];
            pos = s.pos0 + (int32_t)(min(rt * 16 + m, rows - 1) / a.group);  // (columns past the last row: as the last)
        }
        // a row at p sees keys [first_seen(p), p] and those below `first`; hi_m, lo_m: this lane's column, hi_all, lo_all:
        // any row, hi_one, lo_one: every row
        const int32_t edge = (int32_t)s.end - 1, first = (int32_t)min(a.sinks, 1u << 30);
        const int32_t hi_m = min(pos, edge), hi_all = min(phi, edge), hi_one = min(plo, edge);
        const int32_t lo_m = first_seen(pos, a.window), lo_all = first_seen(plo, a.window), lo_one = first_seen(phi, a.window);

        f4 acc[TV];
#pragma unroll
        for (int t = 0; t < TV; ++t) acc[t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        Softmax sm;
#pragma unroll 1
        for (uint32_t t = t0; t < t1; t += 4) {
            const int32_t j0 = (int32_t)tile_at(keys, t) * 32;
            const bool ok0 = here.ok[0], ok1 = here.ok[1], more = t + 4 < t1;
            f4 sv[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
            uint32_t qoff = lane * 16;
            asm volatile("" : "+v"(qoff));  // (the queries stay in LDS: hoisted into registers they make the others spill)
#pragma unroll
            for (int st = 0; st < ST; ++st) {
                if (st % 4 == 0) __builtin_amdgcn_sched_barrier(0);
                const h8 hi = *reinterpret_cast<const h8*>(lds + st * 2048 + qoff), lo = *reinterpret_cast<const h8*>(lds + st * 2048 + 1024 + qoff);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const h8 A = here.k[i].operand(st);
                    sv[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, lo, sv[i], 0, 0, 0);
                    sv[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, hi, sv[i], 0, 0, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if (more) load_k(t + 4, here);
            // a whole tile: every row sees every key
            const bool whole = ok0 & ok1 & (j0 + 31 <= hi_one) & ((j0 >= lo_one) | (j0 + 31 < first));
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int32_t j = j0 + 16 * i + 4 * (int32_t)g + e;
                        const bool in = i ? ok1 : ok0;
                        sv[i][e] = in & (j <= hi_m) & ((j >= lo_m) | (j < first)) ? sv[i][e] : -INFINITY;
                        // keys that no row sees may be anything
                        if (!(in & (j <= hi_all) & ((j >= lo_all) | (j < first)))) here.v[i].clear(e);
                    }
            }
            sm.follow(sv, qs, [&](float f) {
#pragma unroll
                for (int i = 0; i < TV; ++i) acc[i] *= f;
            });
            Softmax::Weights w;
            sm.weights(sv, qs, w);
            const h8 bh = w.high(), bl = w.low();
            constexpr int N = TV < 8 ? TV : 8;
#pragma unroll
            for (int o = 0; o < TV / N; ++o) {
                __builtin_amdgcn_sched_barrier(0);
                uint32_t x[N][2], y[N][2];
                here.v[0].template octet<N>(o, x);
                here.v[1].template octet<N>(o, y);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const h8 A = __builtin_bit_cast(h8, v4u{x[e][0], x[e][1], y[e][0], y[e][1]});
                    f4& to = acc[N * o + e];
                    to = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, bl, to, 0, 0, 0);
                    to = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, bh, to, 0, 0, 0);
                }
            }
            if (more) load_v(t + 4, here);
        }
        // (places made again from the thread's number: kept over the loop they spill)
        uint32_t me = threadIdx.x;
        asm volatile("" : "+v"(me));
        const uint32_t tid = me, lane = me & 63, m = me & 15, g = lane >> 4;
        const float lrun = row_total(sm.l);

        // columns whose sums are not finite, or whose scores are far off
        float zero = lrun * 0.0f;
#pragma unroll
        for (int t = 0; t < TV; ++t) zero += (acc[t][0] + acc[t][1] + acc[t][2] + acc[t][3]) * 0.0f;
        uint64_t odd = __ballot(!(zero == 0.0f) | sm.far_off());
        odd = (odd | odd >> 16 | odd >> 32 | odd >> 48) & 0xFFFF;

        // the waves' sums meet in LDS, eight rows at a time
        float* sums = reinterpret_cast<float*>(lds);  // [wave][row of 8][ROW]
        const uint32_t slot = (start * a.group / 16 + seq + rt) * a.kv_heads + h;
        float* parts0 = a.part + (shares.chunks ? (size_t)part0 : (size_t)slot * splits) * 16 * (W + 4);
        float* part = parts0 + (size_t)split * 16 * (W + 4);
        __syncthreads();  // every wave is past its queries
        if (lane < 16) {
            wm[wave][m] = sm.m;
            wl[wave][m] = lrun;
        }
#pragma unroll 1
        for (uint32_t r0 = 0; r0 < nr; r0 += HALFROWS) {
            if (r0) __syncthreads();
            const uint32_t r = m - r0;
            if (r < HALFROWS && m < nr) {
                float* dst = sums + (wave * HALFROWS + r) * ROW;
#pragma unroll
                for (int t = 0; t < TV; t += 4)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        *reinterpret_cast<f4*>(dst + (4 * (t / V::E) + g) * (W == 512 ? SKEW + 4 : SKEW) + V::E * e + t % V::E) =
                            f4{acc[t][e], acc[t + 1][e], acc[t + 2][e], acc[t + 3][e]};
            }
            for (uint32_t bad = (uint32_t)(odd >> r0) & 0xFF; bad; bad &= bad - 1) {
                const uint32_t c = r0 + __builtin_ctz(bad);
                if (c >= nr) break;
                const uint32_t row = rt * 16 + c;
                constexpr int E = W / 64;
                float q[E], o[E], pm, pl2;
                const float* src = a.q + (size_t)(s.first + row / a.group) * a.q_stride + (size_t)(h * a.group + row % a.group) * W;
#pragma unroll
                for (int e = 0; e < E; ++e) q[e] = src[E * lane + e];
                plain_row<W, Q4>(a, keys, t0, t1, 4, seq, h, s.pos0 + (int32_t)(row / a.group), s.end, q, o, pm, pl2);
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int e = 0; e < E; ++e) sums[(wave * HALFROWS + c - r0) * ROW + skewed(E * lane + e)] = o[e];
                if (lane == 0) {
                    wm[wave][c] = pm;
                    wl[wave][c] = pl2;
                }
            }
            __syncthreads();
            for (uint32_t i = tid; i < min((uint32_t)HALFROWS, nr - r0) * (W / 4); i += 256) {
                const uint32_t c = i / (W / 4), x = i % (W / 4) * 4, row = rt * 16 + r0 + c;
                float M = -INFINITY, L = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; ++w) M = fmaxf(M, wm[w][r0 + c]);
                f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float f = wm[w][r0 + c] == -INFINITY && wl[w][r0 + c] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(wm[w][r0 + c] - M);
                    L = fmaf(f, wl[w][r0 + c], L);
                    if (f != 0.0f) o += f * *reinterpret_cast<const f4*>(sums + (w * HALFROWS + c) * ROW + skewed(x));
                }
                if (parts == 1) {
                    float* out = a.out + (size_t)(s.first + row / a.group) * a.out_stride + (size_t)(h * a.group + row % a.group) * W;
                    *reinterpret_cast<f4*>(out + x) = L == 0.0f ? f4{0.0f, 0.0f, 0.0f, 0.0f} : o / L;
                } else {  // through to the memory side, where the last block finds them
                    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(part, 0, 16 * (W + 4) * 4, 0x00020000);
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, o), rs, ((r0 + c) * (W + 4) + x) * 4, 0, kPartSC1);
                    if (x == 0)
                        __builtin_amdgcn_raw_buffer_store_b64(u2{__float_as_uint(M), __float_as_uint(L)}, rs,
                                                              ((r0 + c) * (W + 4) + W) * 4, 0, kPartSC1);
                }
            }
        }
        if (parts > 1 && !join_apart && last_chunk(a, slot, parts))
            join_parts<W, 1>(a, parts0, parts, 16, 0, nr, rt * 16, s.first, h);
    }
}

// The sequence, its span and the row tile (of R rows) of a partial-sum slot.
__device__ __forceinline__ uint32_t slot_sequence(const PagedAttn& a, uint32_t slot, uint32_t R, uint32_t& tile, Span& s) {
    auto base = [&](uint32_t start, uint32_t k) { return (uint32_t)((uint64_t)min(start, a.b.tokens) * a.group / R) + k; };
    const uint32_t seq = find_span(a.b, [&](uint32_t start, uint32_t k) { return base(start, k) <= slot; }, s, [] {});
    tile = slot - min(slot, base(s.first, seq));
    return seq;
}

// Joins the chunks of (row tile, KV head) slots, a block per 4 / S rows, so that wide tiles of many chunks are read by
// many CUs.
template <int W, int S>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttn a, uint32_t splits, uint32_t chunk, uint32_t R, Shares shares) {
    const uint32_t groups = R * S / 4, slot = blockIdx.x / groups, c0 = blockIdx.x % groups * (4 / S), h = slot % a.kv_heads;
    uint32_t tile;
    Span s;
    const float* part = a.part + (size_t)slot * splits * R * (W + 4);
    if (shares.chunks) {
        Share o;  // (the last sequence whose slots begin at or before this one)
        const uint32_t at = slot / a.kv_heads;
        if (!share(a, shares, R, o, [&](uint32_t, const Span& s, uint32_t first, uint32_t end) {
                const uint32_t base = s.first * a.group / R + (threadIdx.x & 63);
                return end > first && at >= base && at < base + (s.count * a.group + R - 1) / R;
            }))
            return;
        s = o.s;
        chunk = o.chunk;
        splits = kMaxParts;
        tile = at - (o.s.first * a.group / R + o.seq);
        part = a.part + (size_t)(h * shares.chunks + o.first + tile * o.parts) * R * (W + 4);
    } else {
        slot_sequence(a, slot / a.kv_heads, R, tile, s);
    }
    const uint32_t rows = s.count * a.group;
    if (tile * R >= rows) return;
    const uint32_t nr = min(R, rows - tile * R);
    if (c0 >= nr) return;
    const int32_t plo = s.pos0 + (int32_t)(tile * R / a.group), phi = s.pos0 + (int32_t)((tile * R + nr - 1) / a.group);
    const Tiles keys = tiles_of<32>(plo, phi, s.end, a.window, a.sinks);
    uint32_t len, parts;
    chunks_of(keys.count, chunk, splits, len, parts);
    if (parts == 1) return;
    join_parts<W, S>(a, part, parts, R, c0, min(nr, c0 + 4 / S), tile * R, s.first, h);
}

// ---- attention of many rows: drafts, prompts and further turns -------------------------------------------
//
// Row tiles of 64 rows: a wave holds 16 of them from scores to output, their queries and sums in registers, and
// the block's four waves share K and V through LDS, 32 keys at a time in two buffers: while one tile is used, the next
// one is on its way (in registers, then in the other buffer) and one barrier separates tiles.  Bound by the matrix
// cores' 8 W operations per (row, key): both operands' pairs double the 4 W of the two products.  Eight chunks of 512
// tokens at 4,096 positions (16 heads of 256): 530 us fp16, 560 4-bit, 960 TFLOP/s of pairs, 0.89 of what a large
// fp16 product reaches here; one prompt of 512, whose blocks take 8 tiles each, 22 us and 8 the join.
// Slower: 32 rows a wave (one wave a SIMD: 763 us against 586 at that step), the last chunk's block joining (152 against
// 111 us for one chunk of 512).
//
// K lies in LDS as the first product reads it, piece ((half, step), lane) of 16 bytes; V transposed, piece (tile of 16
// channels, lane), its channels ordered by their place in an octet (E values of a load), so that both what a wave
// reads and what it writes are consecutive.  4-bit blocks become fp16 on the way.

template <int W, bool Q4>
__global__ __launch_bounds__(256, W == 512 ? 1 : W >= 128 ? 2 : 4) void paged_many_kernel(PagedAttn a, uint32_t slots, uint32_t splits,
                                                                                          uint32_t chunk, Shares shares) {
    constexpr int ST = W / 32, TV = W / 16, R = kManyRows;
    constexpr int E = W / 16 < 8 ? W / 16 : 8;  // channels of an octet
    constexpr int NK = Q4 ? (W + 255) / 256 : W / 64;  // a thread's pieces of K: blocks of 32 values, or octets
    constexpr int NV = (W + 255) / 256;                // and of V: four keys of an octet of channels
    __shared__ __align__(16) uint8_t lds[2][2][W * 64];  // [buffer][K, V]
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = wave_id(), m = lane & 15, g = lane >> 4;
    uint32_t h, split, rt, seq;
    Span s;
    float* part = a.part;  // the chunk's partial sums
    if (shares.chunks) {
        h = blockIdx.x % a.kv_heads;
        const uint32_t b = blockIdx.x / a.kv_heads;
        Share o;
        if (!share(a, shares, R, o, [&](uint32_t, const Span&, uint32_t first, uint32_t end) { return b >= first && b < end; })) return;
        seq = o.seq;
        s = o.s;
        chunk = o.chunk;
        splits = kMaxParts;
        const uint32_t r = (s.count * a.group + R - 1) / R;
        split = __builtin_amdgcn_readfirstlane(quotient(b - o.first, r));
        rt = r - 1 - (b - o.first - split * r);  // (the last rows, which see the most keys, first)
        part += (size_t)(h * shares.chunks + o.first + rt * o.parts + split) * R * (W + 4);
    } else {
        // blocks b and b + 8 share an XCD: with heads times splits a multiple of 8, a head's row tiles share an L2
        const uint32_t heads = a.kv_heads * splits;
        uint32_t hs, slot;
        if (heads % 8 == 0) {
            hs = blockIdx.x / 8 / slots * 8 + blockIdx.x % 8;
            slot = blockIdx.x / 8 % slots;
        } else {
            hs = blockIdx.x / slots;
            slot = blockIdx.x % slots;
        }
        slot = slots - 1 - slot;  // (a sequence's last rows, which see the most keys, first)
        h = hs % a.kv_heads;
        split = hs / a.kv_heads;
        seq = slot_sequence(a, slot, R, rt, s);
        part += ((size_t)(slot * a.kv_heads + h) * splits + split) * R * (W + 4);
    }
    const uint32_t rows = s.count * a.group;
    if (rt * R >= rows) return;
    const uint32_t nr = min((uint32_t)R, rows - rt * R);
    const int32_t plo = s.pos0 + (int32_t)(rt * R / a.group), phi = s.pos0 + (int32_t)((rt * R + nr - 1) / a.group);
    const Tiles keys = tiles_of<32>(plo, phi, s.end, a.window, a.sinks);
    uint32_t len, parts;
    chunks_of(keys.count, chunk, splits, len, parts);
    if (split >= parts) return;
    const uint32_t t0 = split * len, t1 = min(t0 + len, keys.count);
    const int32_t edge = (int32_t)s.end - 1, first = (int32_t)min(a.sinks, 1u << 30);
    const int32_t hi_all = min(phi, edge), lo_all = first_seen(plo, a.window);

    HalfTable<W, Q4> where;
    // where a tile's halves lie (the last tile again past the end), and whether they have a page
    struct Ref {
        uint64_t off0, off1;
        uint32_t scales0, scales1;
        int32_t j0;
        uint32_t ok;  // bits 0 and 1
    };
    auto ref = [&](uint32_t t) {
        t = min(t, t1 - 1);
        if (t >= where.first + 32) where.fill(a, keys, seq, h, t, 1, t1);
        const uint32_t l = (t - where.first) * 2;
        return Ref{where.offset(l), where.offset(l + 1), where.scales_at(l), where.scales_at(l + 1), (int32_t)tile_at(keys, t) * 32,
                   (uint32_t)(where.ok >> l) & 3};
    };
    // The next tile's K and V on their way.  Thread: pieces of K tid + 256 i, in LDS order (octets: half, step, lane; 4-bit
    // blocks: half, block, row), their addresses scalar plus a constant per lane where a half's share is whole waves
    // (UK); of V: four keys 4 u .. 4 u + 3 of a half, octet o of channels, so that 32 lanes write 256 bytes of LDS in a row.
    constexpr uint32_t PK = Q4 ? W : W * 4;  // pieces of K
    constexpr bool UK = PK / 2 >= 64;
    v4u kr[NK];
    uint32_t kd[Q4 ? NK : 1];
    uint32_t vr[NV][4][Q4 ? 1 : 4], vd[Q4 ? NV : 1][4];
    auto v_piece = [](uint32_t e, uint32_t& half, uint32_t& u, uint32_t& o) {
        constexpr uint32_t O = W / 8 < 16 ? W / 8 : 16;
        half = e / O % 2;
        u = e / (2 * O) % 4;
        o = e / (8 * O) * O + e % O;
    };
    auto load_k = [&](const Ref& r) {
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const uint32_t half = ((UK ? wave * 64 : tid) + 256 * i) / (PK / 2), e = (tid + 256 * i) % (PK / 2);
            const uint8_t* p = a.k_pages + (r.off0 + (half ? r.off1 - r.off0 : 0));
            if constexpr (!Q4) {
                const uint32_t st = UK ? (wave * 64 + 256 * i) % (PK / 2) / 64 : e / 64;
                const auto* q = gp(p) + (st * 64 + m * (W * 2) + g * 16);
                kr[i] = *(const __attribute__((address_space(1))) v4u*)q;
            } else if (PK >= 256 || tid < PK) {
                const auto* q = gp(p) + (e % 16 * (W / 2) + e / 16 * 16);
                const auto* d = gp(p + (r.scales0 + (half ? r.scales1 - r.scales0 : 0))) + (e % 16 * (W / 16) + e / 16 * 2);
                kr[i] = *(const __attribute__((address_space(1))) v4u*)q;
                kd[i] = *(const __attribute__((address_space(1))) uint16_t*)d;
            }
        }
    };
    auto load_v = [&](const Ref& r) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (W < 256 && tid >= W) break;
            uint32_t half, u, o;
            v_piece(tid + 256 * i, half, u, o);
            const uint8_t* p = a.v_pages + (r.off0 + (half ? r.off1 - r.off0 : 0));
            const uint32_t scales = r.scales0 + (half ? r.scales1 - r.scales0 : 0);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if constexpr (!Q4) {
                    const auto* q = gp(p) + (u * (W * 8) + o * 16 + j * (W * 2));
                    const v4u x = *(const __attribute__((address_space(1))) v4u*)q;
                    vr[i][j][0] = x.x, vr[i][j][1] = x.y, vr[i][j][2] = x.z, vr[i][j][3] = x.w;
                } else {
                    const auto* q = gp(p) + (u * (W * 2) + o * 4 + j * (W / 2));
                    const auto* d = gp(p + scales) + (u * (W / 4) + o / 4 * 2 + j * (W / 16));
                    vr[i][j][0] = *(const __attribute__((address_space(1))) uint32_t*)q;
                    vd[i][j] = *(const __attribute__((address_space(1))) uint16_t*)d;
                }
        }
    };
    // the tile into LDS, in slices: KS of K (one write each), then VS of V (4-bit: a key's octet unpacked; then a channel
    // of four keys written)
    constexpr int KS = Q4 ? 4 * NK : NK, VU = Q4 ? 4 : 0, VS = NV * (VU + 8);
    auto store_k = [&](int k, uint8_t* kl) {
        if constexpr (!Q4) {
            *reinterpret_cast<v4u*>(kl + (tid + 256 * k) * 16) = kr[k];
        } else if (PK >= 256 || tid < PK) {
            const uint32_t e = tid + 256 * (k / 4);
            h2 x[4];
            unpack4(kr[k / 4][k % 4], __builtin_bit_cast(_Float16, (uint16_t)kd[k / 4]), x);
            *reinterpret_cast<v4u*>(kl + (e / 16 * 64 + k % 4 * 16 + e % 16) * 16) =
                v4u{__builtin_bit_cast(uint32_t, x[0]), __builtin_bit_cast(uint32_t, x[1]),
                    __builtin_bit_cast(uint32_t, x[2]), __builtin_bit_cast(uint32_t, x[3])};
        }
    };
    // values of keys that no row sees may be anything
    auto clear_v = [&](const Ref& r) {
        if (!((r.ok == 3) & (r.j0 + 31 <= hi_all) & ((r.j0 >= lo_all) | (r.j0 + 31 < first))))
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                uint32_t half, u, o;
                v_piece(tid + 256 * i, half, u, o);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int32_t key = r.j0 + (int32_t)(half * 16 + u * 4) + j;
                    if (!((r.ok >> half & 1) & (key <= hi_all) & ((key >= lo_all) | (key < first)))) {
#pragma unroll
                        for (int x = 0; x < (Q4 ? 1 : 4); ++x) vr[i][j][x] = 0;
                        if constexpr (Q4) vd[i][j] = 0;
                    }
                }
            }
    };
    uint32_t vx[4][4];
    auto store_v = [&](int k, uint8_t* vl) {
        if (W < 256 && tid >= W) return;
        const int i = k / (VU + 8);
        k %= VU + 8;
        if (k < VU) {
            h2 y[4];
            unpack4(vr[i][k][0], __builtin_bit_cast(_Float16, (uint16_t)vd[i][k]), y);
#pragma unroll
            for (int r = 0; r < 4; ++r) vx[k][r] = __builtin_bit_cast(uint32_t, y[r]);
            return;
        }
        // channel 8 o + d: row r = (d % E) W / E + (8 o + d) / E of the transposed tile; its eight-key piece u, half `half`
        const int d = k - VU;
        uint32_t half, u, o;
        v_piece(tid + 256 * i, half, u, o);
        const uint32_t r = o * (8 / E), sel = d & 1 ? 0x07060302u : 0x05040100u;
        uint32_t x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = Q4 ? vx[j][d / 2] : vr[i][j][Q4 ? 0 : d / 2];
        *reinterpret_cast<u2*>(vl + (r / 16 * 1024 + r % 16 * 16 + u * 256 + half * 8) + (d % E) * (W / E) * 64 + d / E * 16) =
            u2{__builtin_amdgcn_perm(x[1], x[0], sel), __builtin_amdgcn_perm(x[3], x[2], sel)};
    };
    auto store = [&](int k, uint8_t* kl, uint8_t* vl) {
        if (k < KS)
            store_k(k, kl);
        else
            store_v(k - KS, vl);
    };
    Ref now, next, after;
    if (t0 < t1) {
        where.fill(a, keys, seq, h, t0, 1, t1);
        now = ref(t0);
        load_k(now);
        load_v(now);
    }

    // the queries: lane (column m, g) holds channels 32 s + 8 g .. + 7 of step s, as scaled fp16 pairs
    h8 qh[ST], ql[ST];
    float qs;
    const uint32_t row0 = rt * R + wave * 16, row = row0 + m, real = min(row, rows - 1);  // (columns past the last row: as the last)
    const int32_t pos = s.pos0 + (int32_t)(real / a.group);
    {
        const float* src = a.q + (size_t)(s.first + real / a.group) * a.q_stride + (size_t)(h * a.group + real % a.group) * W + 8 * g;
        float mx = 0.0f;
#pragma unroll
        for (int st = 0; st < ST; ++st)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const f4 x = *gp(reinterpret_cast<const f4*>(src + 32 * st + 4 * i));
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fabsf(x[e]));
            }
        const float up = pair_scale(lanes4_max(mx));
        qs = a.scale / up * kLog2e;
#pragma unroll
        for (int st = 0; st < ST; ++st)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const f4 x = *gp(reinterpret_cast<const f4*>(src + 32 * st + 4 * i));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float y = x[e] * up;
                    qh[st][4 * i + e] = (_Float16)y;
                    ql[st][4 * i + e] = (_Float16)(y - (float)qh[st][4 * i + e]);
                }
            }
    }
    const bool idle = row0 >= rows;
    const int32_t wlo = s.pos0 + (int32_t)(min(row0, rows - 1) / a.group);
    const int32_t whi = s.pos0 + (int32_t)(min(row0 + 15, rows - 1) / a.group);
    const int32_t hi_one = min(wlo, edge), lo_one = first_seen(whi, a.window);  // (what every one of its rows sees)
    const int32_t hi_m = min(pos, edge), lo_m = first_seen(pos, a.window);

    f4 acc[TV];
    Softmax sm;
#pragma unroll
    for (int t = 0; t < TV; ++t) acc[t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    // S^T of a tile, from its K in LDS; piece(k) does the k-th of eight slices of other work meanwhile
    constexpr int AHEAD = W == 512 ? 3 : 2;  // operands requested ahead of their two products
    auto scores = [&](const uint8_t* kl, f4 (&sv)[2], auto piece) {
        auto at = [&](int f) { return *reinterpret_cast<const h8*>(kl + ((f % 2 * ST + f / 2) * 64 + lane) * 16); };
        sv[0] = sv[1] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        h8 A[2 * ST];
#pragma unroll
        for (int f = 0; f < AHEAD; ++f) A[f] = at(f);
#pragma unroll
        for (int f = 0; f < 2 * ST; ++f) {
            if (f + AHEAD < 2 * ST) A[f + AHEAD] = at(f + AHEAD);
            sv[f % 2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A[f], ql[f / 2], sv[f % 2], 0, 0, 0);
            sv[f % 2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A[f], qh[f / 2], sv[f % 2], 0, 0, 0);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k * ST / 4 == f) piece(k);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    f4 sv[2];
    // the scores of tile `now`: masked where not every row sees every key, the softmax's reference brought along
    auto enter = [&] {
        if (!((now.ok == 3) & (now.j0 + 31 <= hi_one) & ((now.j0 >= lo_one) | (now.j0 + 31 < first))))
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int32_t j = now.j0 + 16 * i + 4 * (int32_t)g + e;
                    sv[i][e] = (now.ok >> i & 1) & (j <= hi_m) & ((j >= lo_m) | (j < first)) ? sv[i][e] : -INFINITY;
                }
        sm.follow(sv, qs, [&](float f) {
#pragma unroll
            for (int v = 0; v < TV; ++v) acc[v] *= f;
        });
    };
    if constexpr (W >= 256) {
        // K is one tile ahead of V: while tile t's weights are taken, tile t + 1's scores are computed, and while V of t is
        // multiplied, K of t + 2 and V of t + 1 go to LDS.  The order of the instructions is the source's, a few at a time:
        // LDS operands requested AHEAD, other work behind each operand's two products (left to itself the compiler
        // requests each operand where it is needed and keeps the products apart from the rest).
        if (t0 < t1) {
#pragma unroll
            for (int k = 0; k < KS; ++k) store_k(k, lds[0][0]);
            clear_v(now);
#pragma unroll
            for (int k = 0; k < VS; ++k) store_v(k, lds[0][1]);
            next = ref(t0 + 1);
            load_k(next);
            load_v(next);
            __syncthreads();
            scores(lds[0][0], sv, [](int) {});
#pragma unroll
            for (int k = 0; k < KS; ++k) store_k(k, lds[1][0]);
            after = ref(t0 + 2);
            load_k(after);
        }
        __syncthreads();
#pragma unroll 1
        for (uint32_t t = t0, b = 0; t < t1; ++t, b ^= 1) {
            Softmax::Weights w;
            f4 ahead[2];
            if (!idle) {
                enter();
                __builtin_amdgcn_sched_barrier(0);
                scores(lds[b ^ 1][0], ahead, [&](int k) { sm.slice(k, sv, qs, w); });
            }
            clear_v(next);
            __builtin_amdgcn_sched_barrier(0);
            if (!idle) {
                const h8 bh = w.high(), bl = w.low();
                const uint8_t* vl = lds[b][1];
                auto at = [&](int v) { return *reinterpret_cast<const h8*>(vl + (v * 64 + lane) * 16); };
                h8 A[TV];
#pragma unroll
                for (int v = 0; v < AHEAD; ++v) A[v] = at(v);
#pragma unroll
                for (int v = 0; v < TV; ++v) {
                    if (v + AHEAD < TV) A[v + AHEAD] = at(v + AHEAD);
                    acc[v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A[v], bl, acc[v], 0, 0, 0);
                    acc[v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A[v], bh, acc[v], 0, 0, 0);
#pragma unroll
                    for (int k = 0; k < KS + VS; ++k)
                        if (k * TV / (KS + VS) == v) store(k, lds[b][0], lds[b ^ 1][1]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                sv[0] = ahead[0];
                sv[1] = ahead[1];
            } else {
#pragma unroll
                for (int k = 0; k < KS + VS; ++k) store(k, lds[b][0], lds[b ^ 1][1]);
            }
            load_v(after);
            now = next;
            next = after;
            after = ref(t + 3);
            load_k(after);
            __syncthreads();
        }
    } else {
        // (narrow heads: few products a tile; more waves per SIMD overlap them better than one wave's own order)
        if (t0 < t1) {
#pragma unroll
            for (int k = 0; k < KS + VS; ++k) {
                if (k == KS) clear_v(now);
                store(k, lds[0][0], lds[0][1]);
            }
            next = ref(t0 + 1);
            load_k(next);
            load_v(next);
        }
        __syncthreads();
#pragma unroll 1
        for (uint32_t t = t0, b = 0; t < t1; ++t, b ^= 1) {
            if (!idle) {
                const uint8_t *kl = lds[b][0] + lane * 16, *vl = lds[b][1] + lane * 16;
                sv[0] = sv[1] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int f = 0; f < 2 * ST; ++f) {
                    const int i = f & 1, st = f >> 1;
                    const h8 A = *reinterpret_cast<const h8*>(kl + (i * ST + st) * 1024);
                    sv[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, ql[st], sv[i], 0, 0, 0);
                    sv[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, qh[st], sv[i], 0, 0, 0);
                }
                enter();
                Softmax::Weights w;
                sm.weights(sv, qs, w);
                const h8 bh = w.high(), bl = w.low();
#pragma unroll
                for (int v = 0; v < TV; ++v) {
                    const h8 A = *reinterpret_cast<const h8*>(vl + v * 1024);
                    acc[v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, bl, acc[v], 0, 0, 0);
                    acc[v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, bh, acc[v], 0, 0, 0);
                }
            }
            if (t + 1 < t1) {
                clear_v(next);
#pragma unroll
                for (int k = 0; k < KS + VS; ++k) store(k, lds[b ^ 1][0], lds[b ^ 1][1]);
                now = next;
                next = ref(t + 2);
                load_k(next);
                load_v(next);
            }
            __syncthreads();
        }
    }
    if (idle) return;

    // rows to the output, or to the chunk's partial sums
    const float l = row_total(sm.l);
    float zero = l * 0.0f;
#pragma unroll
    for (int t = 0; t < TV; ++t) zero += (acc[t][0] + acc[t][1] + acc[t][2] + acc[t][3]) * 0.0f;
    uint64_t odd = __ballot(!(zero == 0.0f) | sm.far_off());
    odd = (odd | odd >> 16 | odd >> 32 | odd >> 48) & 0xFFFF;  // columns whose sums are not finite, or whose scores are far off
    if (row < rows && !(odd >> m & 1)) {
        float* out = a.out + (size_t)(s.first + row / a.group) * a.out_stride + (size_t)(h * a.group + row % a.group) * W;
        float* dst = parts == 1 ? out : part + (row - rt * R) * (W + 4);
        const float f = parts > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
        // tile t's row 4 g + e is row 16 t + 4 g + e of the transposed tile: channel E (it % (W / E)) + it / (W / E)
        constexpr int P = W / E / 16;  // tiles per place in an octet
#pragma unroll
        for (int t = 0; t < P; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int d = 0; d < E; d += 4)
                    *reinterpret_cast<f4*>(dst + E * (16 * t + 4 * g + e) + d) =
                        f4{acc[d * P + t][e], acc[(d + 1) * P + t][e], acc[(d + 2) * P + t][e], acc[(d + 3) * P + t][e]} * f;
        if (parts > 1 && g == 0) *reinterpret_cast<float2*>(dst + W) = make_float2(sm.m, l);
    }
    for (uint32_t bad = (uint32_t)odd; bad; bad &= bad - 1) {
        const uint32_t r = row0 + __builtin_ctz(bad);
        if (r >= rows) break;
        constexpr int EL = W / 64;
        float q[EL], o[EL], pm, pl;
        const size_t at = (size_t)(h * a.group + r % a.group) * W + EL * lane, token = s.first + r / a.group;
#pragma unroll
        for (int e = 0; e < EL; ++e) q[e] = a.q[token * a.q_stride + at + e];
        plain_row<W, Q4>(a, keys, t0, t1, 1, seq, h, s.pos0 + (int32_t)(r / a.group), s.end, q, o, pm, pl);
        float* dst = parts == 1 ? a.out + token * a.out_stride + at : part + (r - rt * R) * (W + 4) + EL * lane;
#pragma unroll
        for (int e = 0; e < EL; ++e) dst[e] = parts > 1 ? o[e] : pl == 0.0f ? 0.0f : o[e] / pl;
        if (parts > 1 && lane == 0) {
            part[(r - rt * R) * (W + 4) + W] = pm;
            part[(r - rt * R) * (W + 4) + W + 1] = pl;
        }
    }
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
    // four rows a wave where they still fill the chip: 256 CUs of 32 waves
    const uint32_t heads = a.q_heads + 2 * a.kv_heads;
    const bool four = (uint64_t)a.b.tokens * heads >= 4 * 8192;
    const uint32_t per = four ? 16 : 4, groups = (heads + per - 1) / per, tasks = a.b.tokens * groups;
    return by_layout(width, q4, [&](auto w, auto t) {
        constexpr int W = decltype(w)::value;
        constexpr bool Q4 = decltype(t)::value;
        const dim3 grid(min(tasks, 1u << 20)), block(256);
        if (four)
            hipLaunchKernelGGL((kv_append_kernel<W, Q4, 4>), grid, block, 0, s, a, groups, tasks);
        else
            hipLaunchKernelGGL((kv_append_kernel<W, Q4, 1>), grid, block, 0, s, a, groups, tasks);
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

hipError_t launch_paged_attention(const PagedAttn& a, uint32_t width, bool q4, const AttnPlan& p, hipStream_t s) {
    return by_layout(width, q4, [&](auto w, auto t) {
        constexpr int W = decltype(w)::value;
        constexpr bool Q4 = decltype(t)::value;
        const dim3 grid(p.shares.chunks ? p.shares.chunks * a.kv_heads : p.units * p.splits), block(256);
        if (p.rows == 16) {
            hipLaunchKernelGGL((p.row_tiles == 1 ? paged_few_kernel<W, Q4, !Q4> : paged_few_kernel<W, Q4, false>), grid, block, 0, s, a,
                               p.units, p.shares.chunks ? kMaxParts : p.splits, p.shares.chunks ? p.slots : p.row_tiles, p.chunk,
                               p.join_apart, p.shares);
        } else {
            hipLaunchKernelGGL((paged_many_kernel<W, Q4>), grid, block, 0, s, a, p.slots, p.splits, p.chunk, p.shares);
        }
        hipError_t e = hipGetLastError();
        if (e == hipSuccess && p.join_apart) {
            // (few rows have many chunks: read by all waves of a block.  52 chunks of 512-wide heads took 12 us by one, 7 by four)
            const uint32_t waves = p.rows == 16 ? 4 : 1;
            hipLaunchKernelGGL((waves == 4 ? paged_join_kernel<W, 4> : paged_join_kernel<W, 1>),
                               dim3(p.slots * a.kv_heads * (p.rows * waves / 4)), block, 0, s, a, p.splits, p.chunk, p.rows, p.shares);
            e = hipGetLastError();
        }
        return e;
    });
}

}  // namespace af
