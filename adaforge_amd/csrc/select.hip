// The choice of a token: penalties, biases and grammar masks on rows of logits, and each row's largest.
//
// One pass over the logits: a block takes a slice of a row, counts the row's history that falls into its slice in
// LDS, and streams the logits through; tokens that neither history nor biases name cost a compare.  A pass is bound
// by its 8 bytes per token (4 without an output).
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

template <bool VEC>
__global__ __launch_bounds__(256) void logits_select_kernel(LogitsSelect a) {
    extern __shared__ uint32_t named[];  // per token of the slice: history count | (bias index + 1) << 16
    __shared__ uint64_t best[4];
    __shared__ uint32_t worst[4], last;
    const uint32_t row = blockIdx.x / a.slices, part = blockIdx.x % a.slices, tid = threadIdx.x;
    const uint32_t base = part * a.slice, n = min(a.slice, a.vocabulary - base);
    for (uint32_t i = tid; i < a.slice; i += 256) named[i] = 0;
    __syncthreads();
    double rep = 1.0, pres = 0.0, freq = 0.0;
    if (a.penalties && a.history) {
        rep = a.penalties[3 * row];
        pres = a.penalties[3 * row + 1];
        freq = a.penalties[3 * row + 2];
        const uint32_t len = min(a.history_len[row], a.history_stride);
        const uint32_t* h = a.history + (size_t)row * a.history_stride;
        for (uint32_t i = tid; i < len; i += 256) {
            const uint32_t t = h[i] - base;
            if (t < n) atomicAdd(&named[t], 1u);
        }
    }
    __syncthreads();
    const float* bv = nullptr;
    if (a.bias_ids) {
        // an id's last bias counts: the largest index (the count below it is the same for all of the id's)
        const uint32_t len = min(a.bias_len[row], a.bias_stride);
        const uint32_t* ids = a.bias_ids + (size_t)row * a.bias_stride;
        bv = a.bias_values + (size_t)row * a.bias_stride;
        for (uint32_t i = tid; i < len; i += 256) {
            const uint32_t t = ids[i] - base;
            if (t < n) atomicMax(&named[t], (i + 1) << 16 | (named[t] & 0xFFFFu));
        }
    }
    __syncthreads();
    const float* x = a.logits + (size_t)row * a.stride + base;
    float* y = a.out ? a.out + (size_t)row * a.out_stride + base : nullptr;
    const uint32_t* mask = a.mask ? a.mask + (size_t)row * a.mask_stride : nullptr;
    uint64_t top = 0;
    uint32_t bad = 0;
    auto one = [&](float v, uint32_t i, uint32_t allow) {
        const uint32_t w = named[i];
        if (w) {
            double d = v;
            if (w & 0xFFFFu) d = (d > 0.0 ? d / rep : d * rep) - __dadd_rn(__dmul_rn(freq, (double)(w & 0xFFFFu)), pres);
            if (w >> 16) d += (double)bv[(w >> 16) - 1];
            v = (float)d;
        }
        if (!allow) v = -INFINITY;
        const uint64_t key = (uint64_t)order_of(v) << 32 | (uint32_t)~(base + i);
        top = key > top ? key : top;
        bad |= !(v < INFINITY);
        return v;
    };
    if constexpr (VEC) {
        for (uint32_t i = 4 * tid; i < n; i += 1024) {
            float v[4];
            const bool whole = i + 4 <= n;
            if (whole) {
                const float4 f = *reinterpret_cast<const float4*>(x + i);
                v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
            } else {
                for (uint32_t e = 0; e < 4; ++e) v[e] = i + e < n ? x[i + e] : -INFINITY;
            }
            const uint32_t bits = mask ? mask[(base + i) / 32] >> ((base + i) % 32) : 0xFu;
            for (uint32_t e = 0; e < 4; ++e)
                if (i + e < n) v[e] = one(v[e], i + e, bits >> e & 1);
            if (y) {
                if (whole)
                    *reinterpret_cast<float4*>(y + i) = make_float4(v[0], v[1], v[2], v[3]);
                else
                    for (uint32_t e = 0; e < 4; ++e)
                        if (i + e < n) y[i + e] = v[e];
            }
        }
    } else {
        for (uint32_t i = tid; i < n; i += 256) {
            const float v = one(x[i], i, mask ? mask[(base + i) / 32] >> ((base + i) % 32) & 1 : 1u);
            if (y) y[i] = v;
        }
    }
    top = wave_best(top);
    const uint64_t any = __ballot(bad);
    if ((tid & 63) == 0) {
        best[tid >> 6] = top;
        worst[tid >> 6] = any != 0;
    }
    __syncthreads();
    // the slices of a row meet at its ticket; the last one in takes the largest of their keys
    const __amdgpu_buffer_rsrc_t prs =
        __builtin_amdgcn_make_buffer_rsrc(a.part + (size_t)row * a.slices, 0, (int)(a.slices * 16), 0x00020000);
    if (tid == 0) {
        for (int w = 1; w < 4; ++w) top = best[w] > top ? best[w] : top;
        bad = worst[0] | worst[1] | worst[2] | worst[3];
        __builtin_amdgcn_raw_buffer_store_b128(v4u{(uint32_t)(top >> 32), (uint32_t)top, bad, 0u}, prs, part * 16, 0, kPartSC1);
        __builtin_amdgcn_s_waitcnt(kWaitVm0);
        last = __hip_atomic_fetch_add(a.tickets + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.slices - 1;
    }
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
        __hip_atomic_store(a.tickets + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

}  // namespace

hipError_t launch_logits_select(const LogitsSelect& a, hipStream_t s) {
    const bool vec = ((uintptr_t)a.logits | (uintptr_t)a.out) % 16 == 0 && a.stride % 4 == 0 && (!a.out || a.out_stride % 4 == 0);
    hipLaunchKernelGGL(vec ? logits_select_kernel<true> : logits_select_kernel<false>, dim3(a.rows * a.slices), dim3(256),
                       a.slice * 4, s, a);
    return hipGetLastError();
}

}  // namespace af
