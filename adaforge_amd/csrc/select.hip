// The choice of a token: penalties, biases and grammar masks on rows of logits, and each row's largest.
//
// One pass over the logits: a block takes a slice of a row, counts the row's history that falls into its slice in
// LDS, and streams the logits through; tokens that neither history nor biases name cost a compare.  A pass is bound
// by its 8 bytes per token (4 without an output): 64 rows of 262,144 with 300 biases and masks 31.5 us = 4.3 TB/s; one row
// by its chain of loads, ticket and last block, 5.9 us.
#include "device.h"
#include "paged.h"

namespace af {

namespace {

constexpr int kPartSC1 = 16;      // buffer access policy sc1: through to (or from) the memory side
constexpr int kWaitVm0 = 0x0F70;  // s_waitcnt vmcnt(0), expcnt and lgkmcnt unconstrained

// A float's order as an unsigned number (-0 as +0); 0 for NaN and -infinity, which are not chosen.
__device__ __forceinline__ uint32_t order_of(float y) {
    if (!(y > -INFINITY)) return 0;
    const uint32_t u = __float_as_uint(y + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint64_t wave_best(uint64_t k) {
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const uint64_t o = __shfl_xor(k, d);
        k = o > k ? o : k;
    }
    return k;
}

// T: threads, which take the slice's tokens by quads; VEC: rows of logits and out are 16-byte aligned.
template <int T, bool VEC>
__global__ __launch_bounds__(T) void logits_select_kernel(LogitsSelect a) {
    constexpr uint32_t SLICE = kLogitsSlice;
    constexpr int Q = SLICE / 4 / T, WAVES = T / 64;  // quads of a thread
    __shared__ __align__(16) uint32_t named[SLICE];  // per token of the slice: history count | (bias index + 1) << 16
    __shared__ uint64_t best[WAVES];
    __shared__ uint32_t worst[WAVES], last;
    const uint32_t row = blockIdx.x / a.slices, part = blockIdx.x % a.slices, tid = threadIdx.x;
    const uint32_t base = part * SLICE, n = min(SLICE, a.vocabulary - base);
    // the slice is on its way while its history is counted: thread's quad q at tokens 4 (T q + tid)
    const float* x = a.logits + (size_t)row * a.stride + base;
    float v[Q][4];
    uint32_t bits[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const uint32_t i = 4 * (T * q + tid);
        if (VEC && i + 4 <= n) {
            const float4 f = *reinterpret_cast<const float4*>(x + i);
            v[q][0] = f.x, v[q][1] = f.y, v[q][2] = f.z, v[q][3] = f.w;
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) v[q][e] = i + e < n ? x[i + e] : -INFINITY;
        }
        bits[q] = a.mask && i < n ? a.mask[(size_t)row * a.mask_stride + (base + i) / 32] : 0xFFFFFFFFu;
    }
    // and so are the row's lists: their first entries whether they count or not
    const bool past = a.penalties && a.history;
    const uint32_t* h = a.history + (size_t)row * a.history_stride;
    const uint32_t* ids = a.bias_ids + (size_t)row * a.bias_stride;
    constexpr int H = 1024 / T, B = T < 512 ? 512 / T : 1;
    uint32_t hist[H], bias[B];
#pragma unroll
    for (int u = 0; u < H; ++u) hist[u] = past && tid + T * u < a.history_stride ? h[tid + T * u] : 0;
#pragma unroll
    for (int u = 0; u < B; ++u) bias[u] = a.bias_ids && tid + T * u < a.bias_stride ? ids[tid + T * u] : 0;
    const uint32_t hist_len = past ? min(a.history_len[row], a.history_stride) : 0;
    const uint32_t bias_len = a.bias_ids ? min(a.bias_len[row], a.bias_stride) : 0;
    double rep = 1.0, pres = 0.0, freq = 0.0;
    if (past) {
        rep = a.penalties[3 * row];
        pres = a.penalties[3 * row + 1];
        freq = a.penalties[3 * row + 2];
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) *reinterpret_cast<uint4*>(named + 4 * (T * q + tid)) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (hist_len) {
        auto count = [&](uint32_t id, uint32_t i) {
            if (i < hist_len && id - base < n) atomicAdd(&named[id - base], 1u);
        };
#pragma unroll
        for (int u = 0; u < H; ++u) count(hist[u], tid + T * u);
        for (uint32_t i0 = tid + T * H; i0 < hist_len; i0 += 4 * T) {
            uint32_t t[4];
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) t[u] = i0 + T * u < hist_len ? h[i0 + T * u] : 0;
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) count(t[u], i0 + T * u);
        }
        __syncthreads();
    }
    const float* bv = a.bias_values + (size_t)row * a.bias_stride;
    if (bias_len) {
        // an id's last bias counts: the largest index (the count below it is the same for all of the id's)
        auto note = [&](uint32_t id, uint32_t i) {
            if (i < bias_len && id - base < n) atomicMax(&named[id - base], (i + 1) << 16 | (named[id - base] & 0xFFFFu));
        };
#pragma unroll
        for (int u = 0; u < B; ++u) note(bias[u], tid + T * u);
        for (uint32_t i = tid + T * B; i < bias_len; i += T) note(ids[i], i);
        __syncthreads();
    }
    float high = -INFINITY;  // of the thread's, its lowest token (they come in rising order)
    uint32_t at = 0;
    bool odd = false;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const uint32_t i = 4 * (T * q + tid);
        const uint4 w4 = *reinterpret_cast<const uint4*>(named + i);
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
        if (w4.x | w4.y | w4.z | w4.w)
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                if (w[e]) {
                    double d = v[q][e];
                    const double c = w[e] & 0xFFFFu;
                    if (w[e] & 0xFFFFu) d = (d > 0.0 ? d / rep : d * rep) - __dadd_rn(__dmul_rn(freq, c), pres);
                    if (w[e] >> 16) d += (double)bv[(w[e] >> 16) - 1];
                    v[q][e] = (float)d;
                }
        const uint32_t allow = bits[q] >> ((base + i) % 32);
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            if (!(allow >> e & 1)) v[q][e] = -INFINITY;
            if (v[q][e] > high) {
                high = v[q][e];
                at = i + e;
            }
            odd |= !(v[q][e] < INFINITY);
        }
    }
    uint64_t top = wave_best((uint64_t)order_of(high) << 32 | (uint32_t)~(base + at));
    uint32_t bad;
    const uint64_t any = __ballot(odd);
    if ((tid & 63) == 0) {
        best[tid >> 6] = top;
        worst[tid >> 6] = any != 0;
    }
    __syncthreads();
    // The slices of a row meet at its ticket; the last one in takes the largest of their keys.  The ticket is drawn
    // before the slice is stored, which it need not wait for.
    const __amdgpu_buffer_rsrc_t prs =
        __builtin_amdgcn_make_buffer_rsrc(a.part + (size_t)row * a.slices, 0, (int)(a.slices * 16), 0x00020000);
    uint32_t ticket = 0;
    if (tid == 0) {
        bad = worst[0];
        for (int w = 1; w < WAVES; ++w) {
            top = best[w] > top ? best[w] : top;
            bad |= worst[w];
        }
        __builtin_amdgcn_raw_buffer_store_b128(v4u{(uint32_t)(top >> 32), (uint32_t)top, bad, 0u}, prs, part * 16, 0, kPartSC1);
        __builtin_amdgcn_s_waitcnt(kWaitVm0);
        ticket = __hip_atomic_fetch_add(a.tickets + row * a.ticket_stride, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (a.out) {
        float* y = a.out + (size_t)row * a.out_stride + base;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const uint32_t i = 4 * (T * q + tid);
            if (VEC && i + 4 <= n)
                *reinterpret_cast<float4*>(y + i) = make_float4(v[q][0], v[q][1], v[q][2], v[q][3]);
            else
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e)
                    if (i + e < n) y[i + e] = v[q][e];
        }
    }
    if (tid == 0) last = ticket == a.slices - 1;
    __syncthreads();
    if (!last || tid >= 64) return;
    top = 0;
    bad = 0;
    for (uint32_t i = tid; i < a.slices; i += 64) {
        const v4u p = __builtin_amdgcn_raw_buffer_load_b128(prs, i * 16, 0, kPartSC1);
        const uint64_t k = (uint64_t)p.x << 32 | p.y;
        top = k > top ? k : top;
        bad |= p.z;
    }
    top = wave_best(top);
    const uint64_t found = __ballot(bad);
    if (tid == 0) {
        a.result[2 * row] = top >> 32 ? ~(uint32_t)top : 0xFFFFFFFFu;
        a.result[2 * row + 1] = found != 0;
        __hip_atomic_store(a.tickets + row * a.ticket_stride, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

}  // namespace

hipError_t launch_logits_select(const LogitsSelect& a, hipStream_t s) {
    const bool vec = ((uintptr_t)a.logits | (uintptr_t)a.out) % 16 == 0 && a.stride % 4 == 0 && (!a.out || a.out_stride % 4 == 0);
    // few blocks: four times the threads, with a quarter of the work each (one row of 262,144 tokens 6.2 us, with 256
    // threads 6.8; 64 rows 32 us, with 1,024 threads 48)
    const dim3 grid(a.rows * a.slices);
    if (grid.x >= 1024)
        hipLaunchKernelGGL((vec ? logits_select_kernel<256, true> : logits_select_kernel<256, false>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((vec ? logits_select_kernel<1024, true> : logits_select_kernel<1024, false>), grid, dim3(1024), 0, s, a);
    return hipGetLastError();
}

}  // namespace af
