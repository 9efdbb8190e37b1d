// cache_attention.cuh -- grouped-query attention of a step's rows over a paged K/V cache.
//
//   o[i, h] = sum_s p_s V[s, h/G],  p = softmax over visible s of scale * q[i, h] . K[s, h/G]
//
// Row i of sequence b sees every committed token (s < base[b]) and node j of its own step
// (s = base[b] + j) when bit j of mask[row] is set, or, without a mask, when j <= i. A row that
// sees nothing gives zero.
#pragma once

#include "cache.cuh"

namespace mica {

struct CacheAttnArgs {
    CachePlan plan;
    const __nv_bfloat16* q;     // [N, ldq] H heads of D
    long ldq;
    const __nv_bfloat16* k_pages;
    const __nv_bfloat16* v_pages;
    long page_stride;           // elements
    const unsigned long long* mask;   // [N, ld_mask] or nullptr (causal)
    long ld_mask;
    int words;                  // 64-bit words of a row's mask
    __nv_bfloat16* out;         // [N, ldo]
    long ldo;
    int H, KV;
    float scale_log2;           // scale * log2(e)
};

// Simplest form: one warp per (row, query head), one key at a time, running maximum and sum.
template <int D>
__global__ void __launch_bounds__(128) cache_attention_kernel(const CacheAttnArgs a) {
    constexpr int E = D / 32;
    const long w = (static_cast<long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (w >= static_cast<long>(a.plan.N) * a.H) return;
    const int row = static_cast<int>(w / a.H), h = static_cast<int>(w % a.H);
    const int kvh = h / (a.H / a.KV);
    const int b = cache_sequence_of(a.plan, row);
    float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q[e] = __bfloat162float(a.q[static_cast<long>(row) * a.ldq + static_cast<long>(h) * D + lane + 32 * e]) * a.scale_log2;
        o[e] = 0.f;
    }
    if (b >= 0) {
        const int base = a.plan.base[b], first = a.plan.cu[b];
        const int rows = min(a.plan.cu[b + 1], a.plan.N) - first;
        bool bad = base < 0;
        for (long s = 0; s < static_cast<long>(base) + rows && !bad; ++s) {
            const long j = s - base;
            if (j >= 0) {
                const bool seen = a.mask ? j < 64l * a.words && (a.mask[row * a.ld_mask + (j >> 6)] >> (j & 63) & 1)
                                         : j <= row - first;
                if (!seen) continue;
            }
            int page, slot;
            if (!cache_slot(a.plan, b, s, &page, &slot)) { bad = true; break; }
            const long off = static_cast<long>(page) * a.page_stride + ((static_cast<long>(kvh) << a.plan.page_log2) + slot) * D;
            float z = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) z += q[e] * __bfloat162float(a.k_pages[off + lane + 32 * e]);
            z = warp_sum(z);
            const float mn = fmaxf(m, z);
            const float al = m == -INFINITY ? 0.f : exp2f(m - mn), p = mn == -INFINITY ? 0.f : exp2f(z - mn);
            l = l * al + p;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = o[e] * al + p * __bfloat162float(a.v_pages[off + lane + 32 * e]);
            m = mn;
        }
        if (bad && lane == 0) record_bad_page();
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
    for (int e = 0; e < E; ++e)
        a.out[static_cast<long>(row) * a.ldo + static_cast<long>(h) * D + lane + 32 * e] = __float2bfloat16_rn(o[e] * inv);
}

}  // namespace mica
