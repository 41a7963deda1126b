// The paged KV cache of several sequences: where a batch's tokens stand, which keys they see, and the kernels'
// arguments.  The index arithmetic compiles for the host too (tests run it there); device arrays may hold anything,
// so every value read from one is cut to range here.
#pragma once
#include <stddef.h>
#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define AF_HD __host__ __device__ __forceinline__
#else
#define AF_HD inline
#endif

namespace af {

struct PagedBatch {
    const uint32_t* starts;
    const uint32_t* lengths;
    const uint32_t* table;
    uint32_t table_stride, sequences, tokens;
    uint32_t pages, page_shift;  // pages of 2^page_shift tokens
};

constexpr int32_t kNoPosition = -(1 << 30);

// A sequence's rows [first, first + count) of the batch, the position of the first, and the keys [0, end) that its
// table can hold.
struct Span {
    uint32_t first, count;
    int32_t pos0;
    uint32_t end;
};

AF_HD Span span_of(uint32_t start, uint32_t stop, uint32_t length, const PagedBatch& b) {
    const uint32_t len = length < (1u << 30) ? length : 1u << 30;
    const uint32_t a = start < b.tokens ? start : b.tokens, e = stop < b.tokens ? stop : b.tokens;
    const uint32_t cap = b.table_stride << b.page_shift;  // (at most 2^24: checked by the call)
    Span s;
    s.first = a;
    s.count = e > a ? e - a : 0;
    const int64_t p = (int64_t)len - ((int64_t)stop - (int64_t)a);
    s.pos0 = s.count && p > kNoPosition ? (int32_t)p : kNoPosition;
    s.end = len < cap ? len : cap;
    return s;
}

// Whether the query at position p sees key j (of those its sequence holds).
AF_HD bool sees(int32_t p, int32_t j, uint32_t window, uint32_t sinks) {
    return j <= p && (window == 0 || (uint32_t)(p - j) < window || (uint32_t)j < sinks);
}

// The key tiles (of T keys) that hold every key seen by queries at positions plo .. phi: tiles [0, head), then from,
// from + 1, ...; `count` in all.
struct Tiles {
    uint32_t head, from, count;
};

template <uint32_t T>
AF_HD Tiles tiles_of(int32_t plo, int32_t phi, uint32_t end, uint32_t window, uint32_t sinks) {
    Tiles t = {0, 0, 0};
    if (phi < 0) return t;
    const uint32_t hi = (uint32_t)phi + 1 < end ? (uint32_t)phi + 1 : end;  // keys [0, hi)
    const uint32_t low = plo < 0 ? 0u : (uint32_t)plo;
    const uint32_t lo = window != 0 && low + 1 > window ? low + 1 - window : 0u;
    const uint32_t to = (hi + T - 1) / T;
    uint32_t first = sinks < lo ? sinks : lo;  // first tokens that the window leaves out
    t.head = (first + T - 1) / T;
    if (t.head > to) t.head = to;
    t.from = lo / T > t.head ? lo / T : t.head;
    t.count = t.head + (to > t.from ? to - t.from : 0);
    return t;
}

AF_HD uint32_t tile_at(const Tiles& t, uint32_t i) { return i < t.head ? i : t.from + (i - t.head); }

// Bytes of one KV head's part of a page.
AF_HD uint32_t page_part_bytes(bool q4, uint32_t page, uint32_t width) {
    return q4 ? page * (width / 16 * 9) : page * width * 2;
}

// A workspace starts with completion tickets, zero between calls; partial results follow.
constexpr uint32_t kTickets = 16384;
constexpr size_t kTicketBytes = kTickets * 4;

// The distance of `count` tickets: up to a cache line of 128 bytes.  The memory side takes the draws of one line in
// turn, about 5 ns each: 4,096 blocks that drew from 64 adjacent words took 20 us for it.
inline uint32_t ticket_stride(uint64_t count) {
    uint32_t s = 32;
    while (s > 1 && count * s > kTickets) s /= 2;
    return s;
}

// What the split of an attention call depends on: sizes, and the caller's hints.
struct AttnShape {
    uint32_t sequences, tokens, kv_heads, group, width, window, sinks;
    uint32_t longest_query, longest_context, capacity;  // (capacity: positions a page table row holds)
    bool q4;
};

// Row tiles' slots for partial sums: sequence s's tiles start at slot starts[s] group / R + s, so every sequence's lie
// in front of the next one's whatever the starts are.
AF_HD uint32_t row_slots(const AttnShape& a, uint32_t r) { return (uint32_t)((uint64_t)a.tokens * a.group / r) + a.sequences; }

AF_HD uint32_t least(uint32_t a, uint32_t b) { return a < b ? a : b; }
AF_HD uint32_t most(uint32_t a, uint32_t b) { return a > b ? a : b; }

// The longest key range of a row tile, in tiles of 32 keys, as the hints have it.
AF_HD uint32_t longest_tiles(const AttnShape& a, uint32_t tokens) {
    uint32_t keys = most(1, least(a.longest_context, a.capacity));
    if (a.window) {
        const uint64_t seen = (uint64_t)a.window + a.sinks + tokens + 64;
        if (seen < keys) keys = (uint32_t)seen;
    }
    return (keys + 31) / 32;
}

constexpr uint32_t kManyRows = 64;

// Chunks shared out by the work there is, not by the longest sequence: up to 64 sequences, whose key tiles every block adds up
// for itself (a lane a sequence).  A KV head's chunks take `chunks` blocks at most (0: shared
// out by the hints), of which those that fill the chip or even out what is left are `most`, and one a row tile
// (`slots`).  32 conversations of 1 to 8,192 positions took 229 us by the longest and take 205 so, eight of 512-wide
// heads 54 and 45, 16 of 64-wide ones 32 and 24; equal lengths lose what the addition costs, about 1 us a block: 16 at
// 8,192 positions 96 and 98.
struct Shares {
    uint32_t most, chunks, slots;
    uint32_t per_fill, per_safe, per_even;  // 2^32 over a number of chunks, rounded up: the blocks divide by multiplying
    uint32_t few, some;                    // key tiles that a chunk has at least, where it fills the chip, and where it evens out
};

// x over the number of chunks (2 or more) that `per` belongs to, rounded up.
AF_HD uint32_t per_chunk(uint32_t x, uint32_t per) { return (uint32_t)(((uint64_t)(x ? x - 1 : 0) * per) >> 32) + 1; }

constexpr uint32_t kMaxParts = 128;

// The key tiles of a chunk where the row tiles' key tiles come to `total`, `fill` chunks fill the chip and `even` even out.
// Chunks of it are at most the larger number and one a row tile.
AF_HD uint32_t share_of(const Shares& s, uint32_t total, uint32_t per_fill) {
    return (least(most(s.few, per_chunk(total, per_fill)), most(s.some, per_chunk(total, s.per_even))) + 3) / 4 * 4;
}

// The chunk of a sequence of n key tiles: its share, but no small rest, and not above kMaxParts chunks.
AF_HD uint32_t share_chunk(uint32_t share, uint32_t n) {
    return n <= share + share / 2 ? most(n, 1) : most(share, (n + kMaxParts - 1) / kMaxParts);
}

// A launch: row tiles of `rows` rows, their keys in at most `splits` chunks of `chunk` tiles or more.  16 rows: grid
// units (row tiles, sequences, KV heads) by splits; more: grid slots, KV heads and splits.
struct AttnPlan {
    uint32_t rows, units, row_tiles, slots, splits, chunk;
    bool join_apart;  // the chunks are joined by a launch of their own
    Shares shares;
    size_t part_bytes;
};

AF_HD AttnPlan attn_plan(const AttnShape& a) {
    AttnPlan p;
    p.shares = Shares{};
    const uint32_t tokens = most(1, least(a.longest_query, a.tokens));
    const uint64_t pairs = (uint64_t)a.sequences * a.kv_heads;  // (at most 2^22: checked by the call)
    const uint32_t tiles = longest_tiles(a, tokens);
    p.row_tiles = (uint32_t)(((uint64_t)tokens * a.group + 15) / 16);
    // Row tiles of 16 read K and V once each, through an L2; tiles of 64 rows share them through LDS, which pays as soon as
    // what is read fills the chip.  With fewer key tiles, from five row tiles on: eight sequences of 300 positions, three
    // row tiles of 256-wide fp16 heads 20 us, by 64 rows 23; of 1,000 in 128-wide heads 21 and 29; 80 rows at 300 22 and 18.
    // With more, from three on: eight of 4,096, three row tiles of 256-wide 4-bit heads 74 and 63, 16 of up to 16,000 in
    // 512-wide heads, four row tiles 148 and 100, fp16 231 and 99.  From two on where a row tile reads most: 512 wide 149 and
    // 77, 4 bits 97 and 79, 256-wide fp16 102 and 77, 128-wide 56 and 46 (but 4 bits 45 and 51, 64-wide 31 and 34).  64-wide
    // 4-bit heads read the least: 100 of 400 to 4,000, three row tiles 149 and 207.
    const uint32_t apart = pairs * tiles <= 2048 || (a.q4 && a.width == 64) ? 4 : a.width == 512 || (!a.q4 && a.width >= 128) ? 1 : 2;
    p.rows = p.row_tiles > apart ? kManyRows : 16;
    p.slots = row_slots(a, p.rows);
    if (p.row_tiles * pairs > 1u << 22) p.row_tiles = most(1, (uint32_t)((1u << 22) / pairs));
    const uint64_t sums = (uint64_t)p.slots * a.kv_heads;
    uint32_t splits;
    if (p.rows == 16) {
        p.units = (uint32_t)(p.row_tiles * pairs);
        // as many chunks as fill the chip, then more of at least 32 tiles for lengths that differ (32 conversations of up
        // to 8,192 positions 205 us, of 64 tiles 217; eight of 512-wide heads 44, of 16 tiles 70)
        const uint32_t fill = least(most(1, 256 / p.units), (tiles + 3) / 4);
        const uint32_t even = least(most(1, 2048 / p.units), most(1, tiles / 32));
        splits = least(most(fill, even), 128);
        splits = sums > kTickets ? 1 : least(splits, most(1, (uint32_t)(8192 / sums)));
    } else {
        p.units = (uint32_t)sums;
        // two blocks a CU (a prompt of 512 rows in chunks of 8 tiles 30 us, of 4 tiles 33), or four of longer chunks
        splits = most(least(most(1, 512 / p.units), most(1, tiles / 8)), least(most(1, 1024 / p.units), most(1, tiles / 16)));
        splits = least(splits, 16);
    }
    p.chunk = (tiles + splits - 1) / splits;
    p.splits = (tiles + p.chunk - 1) / p.chunk;
    const bool one = p.rows == 16;
    const uint32_t row_tiles = one ? p.row_tiles : (uint32_t)(((uint64_t)tokens * a.group + 63) / 64);
    // (of 64 rows where a sequence has few row tiles, and then for one round of blocks: eight sequences of 120 rows at 4,096
    // positions 138 us by the longest and 113 so, of 48 rows at 700 to 8,192 91 and 83; many row tiles even themselves
    // out: four sequences of 258 to 1,024 rows 327 and 332, but 848 and 803 in 512-wide heads, whose blocks have a CU each)
    const bool uneven = one ? a.sequences > 1 && tiles > 4 : p.splits > 1 && (row_tiles <= 4 || a.width == 512);
    if (uneven && a.sequences <= 64 && p.slots <= 512 && sums <= (one ? 2048 : 512)) {
        const uint32_t few = one ? 4 : 8, some = one ? 32 : 16;
        const uint32_t fill = most(2, (one || a.width == 512 ? 256 : 512) / a.kv_heads), safe = most(2, fill - least(fill, p.slots));
        const uint32_t even = one ? most(2, least(2048 / a.kv_heads, a.sequences * row_tiles * tiles / some)) : fill;
        auto per = [](uint32_t n) { return (uint32_t)(((1ull << 32) + n - 1) / n); };
        p.shares = Shares{most(fill, even), most(fill, even) + p.slots, p.slots, per(fill), per(safe), per(even), few, some};
    }
    const uint64_t row_bytes = (uint64_t)(a.width + 4) * 4;
    // (many partial sums are stored, and joined, faster by many blocks of another launch: its partial sums need not go
    // through to the memory side.  A prompt of 512 at 4,096 positions took 152 us joined by the last chunks, 111 apart.)
    p.join_apart = p.splits > 1 && (p.rows > 16 || p.splits * least(16, tokens * a.group) * row_bytes > 131072);
    p.part_bytes = p.splits > 1 ? (size_t)(sums * p.splits * p.rows * row_bytes) : 0;
    if (p.shares.chunks) p.part_bytes = (size_t)((uint64_t)p.shares.chunks * a.kv_heads * p.rows * row_bytes);
    return p;
}

#ifdef __HIPCC__

struct KvAppend {
    const float *q, *k, *v;
    uint32_t q_stride, k_stride, v_stride;
    const float *q_norm, *k_norm;
    float q_eps, k_eps, v_eps;
    uint32_t v_norm;
    const uint64_t* turns;  // per pair, the fraction of a turn per position (null: no rotation)
    uint32_t q_heads, kv_heads;
    float* q_out;
    uint32_t q_out_stride;
    uint8_t *k_pages, *v_pages;
    PagedBatch b;
};
hipError_t launch_kv_append(const KvAppend& a, uint32_t width, bool q4, hipStream_t s);
hipError_t launch_kv_read(const uint8_t* k_pages, const uint8_t* v_pages, const PagedBatch& b, uint32_t kv_heads,
                          uint32_t width, bool q4, uint16_t* k, uint16_t* v, hipStream_t s);

struct PagedAttn {
    const float* q;
    float* out;
    uint32_t q_stride, out_stride;
    const uint8_t *k_pages, *v_pages;
    uint32_t kv_heads, group;  // query heads per KV head
    uint32_t window, sinks;
    float scale;
    PagedBatch b;
    uint32_t* tickets;
    uint32_t ticket_stride;
    float* part;
};
hipError_t launch_paged_attention(const PagedAttn& a, uint32_t width, bool q4, const AttnPlan& plan, hipStream_t s);

struct LogitsSelect {
    const float* logits;
    float* out;
    uint32_t stride, out_stride, rows, vocabulary;
    const float* penalties;
    const uint32_t *history, *history_len;
    uint32_t history_stride;
    const uint32_t* bias_ids;
    const float* bias_values;
    const uint32_t* bias_len;
    uint32_t bias_stride;
    const uint32_t* mask;
    uint32_t mask_stride;
    uint32_t* result;
    uint32_t* tickets;
    uint32_t ticket_stride;
    uint4* part;      // one (key high, key low, bad, 0) per slice of a row
    uint32_t slices;
};
hipError_t launch_logits_select(const LogitsSelect& a, hipStream_t s);

#endif

// Tokens of a row that a block takes in the choice of a token.
constexpr uint32_t kLogitsSlice = 4096;

}  // namespace af
