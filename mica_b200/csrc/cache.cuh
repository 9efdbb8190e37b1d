// cache.cuh -- paged K/V cache: the step plan shared by its kernels, the fused q/k norm +
// rotation + write into the pages, page copies, and the move of accepted tokens.
//
// One layer's pages are bf16 [pages, KV, page, D] (any page stride: the whole pool is
// [pages, layers, 2, KV, page, D]). Sequence b of a step has base[b] committed tokens and the
// step's rows cu[b] .. cu[b+1]; its row i sits at cache index base[b] + i, which is slot
// (index % page) of page table[b][index / page].
//
// Every index read from device memory is checked before it is used: a sequence whose base or rows
// do not fit its table, or a page number outside the pool, records MICA_DEV_BAD_PAGE in the device
// error word and touches no memory.
#pragma once

#include "quant.cuh"

namespace mica {

struct CachePlan {
    const int* table;      // [B, P] page numbers
    long ld_table;
    const int* base;       // [B] committed tokens
    const int* cu;         // [B + 1] first row of each sequence
    int B, P, N;           // sequences, table width, rows of the step's tensors
    int pages;             // pages of the pool
    int page_log2;
};

__device__ __forceinline__ void record_bad_page() { atomicExch(&g_dev_error, MICA_DEV_BAD_PAGE); }

// Sequence of row `row`: the b with cu[b] <= row < cu[b+1], or -1 for a row behind the last
// sequence. Whole-warp search: each level splits the range 32 ways, one load per lane, so 1024
// sequences take two loads in a row.
__device__ __forceinline__ int cache_sequence_of(const CachePlan& p, int row) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = p.B;                       // the answer is the count of ends cu[1..B] <= row
    while (n > 0) {
        const int step = (n + 31) >> 5;
        const int i = lo + min(n, (lane + 1) * step) - 1;
        const bool le = (lane * step < n) && p.cu[i + 1] <= row;
        const int c = __popc(__ballot_sync(0xffffffffu, le));
        const int taken = min(n, c * step);
        lo += taken;
        n = step == 1 ? 0 : min(step - 1, n - taken);
    }
    return lo < p.B && row >= p.cu[lo] ? lo : -1;
}

// Page number and slot of cache index `index` of sequence b; false when it is not in the table or
// the table names no page of the pool.
__device__ __forceinline__ bool cache_slot(const CachePlan& p, int b, long index, int* page, int* slot) {
    const long at = index >> p.page_log2;
    if (index < 0 || at >= p.P) return false;
    const int pg = p.table[static_cast<long>(b) * p.ld_table + at];
    if (pg < 0 || pg >= p.pages) return false;
    *page = pg;
    *slot = static_cast<int>(index & ((1 << p.page_log2) - 1));
    return true;
}

// ---------------------------------------------------------------------------------------
struct AppendArgs {
    CachePlan plan;
    const __nv_bfloat16* qkv;   // [N, ld] rows q (H*D) | k (KV*D) | v (KV*D)
    long ld;
    const __nv_bfloat16* q_w;   // [D]
    const __nv_bfloat16* k_w;   // [D]
    const __nv_bfloat16* cos;   // [n_pos, D]
    const __nv_bfloat16* sin;
    long n_pos;
    const long* pos;            // [N] or nullptr (= cache index)
    __nv_bfloat16* q_out;       // [N, ldq]
    long ldq;
    __nv_bfloat16* k_pages;
    __nv_bfloat16* v_pages;
    long page_stride;           // elements
    int H, KV;
    float eps;
};

// One warp per (row, head): the simplest form.
template <int D>
__global__ void __launch_bounds__(256) cache_append_kernel(const AppendArgs a) {
    constexpr int E = D / 64;                 // pairs (d, d + D/2) per lane
    const long w = (static_cast<long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    const int heads = a.H + 2 * a.KV;
    const long row_l = w / heads;
    if (row_l >= a.plan.N) return;
    const int row = static_cast<int>(row_l), h = static_cast<int>(w % heads);
    const int b = cache_sequence_of(a.plan, row);
    const __nv_bfloat16* x = a.qkv + static_cast<long>(row) * a.ld + static_cast<long>(h) * D;
    __nv_bfloat16* q = a.q_out + static_cast<long>(row) * a.ldq + static_cast<long>(h) * D;
    long index = 0, p = 0;
    bool ok = b >= 0;
    int page = 0, slot = 0;
    if (ok) {
        index = static_cast<long>(a.plan.base[b]) + (row - a.plan.cu[b]);
        ok = a.plan.base[b] >= 0 && cache_slot(a.plan, b, index, &page, &slot);
        p = a.pos ? a.pos[row] : index;
        ok = ok && p >= 0 && p < a.n_pos;
        if (!ok && lane == 0) record_bad_page();
    }
    if (!ok) {
        if (h < a.H)
            for (int d = lane; d < D; d += 32) q[d] = __float2bfloat16_rn(0.f);
        return;
    }
    const int kvh = (h - a.H) % a.KV;
    __nv_bfloat16* kv = (h < a.H + a.KV ? a.k_pages : a.v_pages) + static_cast<long>(page) * a.page_stride +
                        ((static_cast<long>(kvh) << a.plan.page_log2) + slot) * D;
    if (h >= a.H + a.KV) {
        for (int d = lane; d < D; d += 32) kv[d] = x[d];
        return;
    }
    float lo[E], hi[E], ss = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        lo[i] = __bfloat162float(x[lane + 32 * i]);
        hi[i] = __bfloat162float(x[D / 2 + lane + 32 * i]);
        ss += lo[i] * lo[i] + hi[i] * hi[i];
    }
    ss = warp_sum(ss);
    const float r = rsqrtf(ss / static_cast<float>(D) + a.eps);
    const __nv_bfloat16* wt = h < a.H ? a.q_w : a.k_w;
    __nv_bfloat16* o = h < a.H ? q : kv;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int dl = lane + 32 * i, dh = dl + D / 2;
        const float yl = lo[i] * r * __bfloat162float(wt[dl]), yh = hi[i] * r * __bfloat162float(wt[dh]);
        o[dl] = __float2bfloat16_rn(yl * __bfloat162float(a.cos[p * D + dl]) - yh * __bfloat162float(a.sin[p * D + dl]));
        o[dh] = __float2bfloat16_rn(yh * __bfloat162float(a.cos[p * D + dh]) + yl * __bfloat162float(a.sin[p * D + dh]));
    }
}

// ---------------------------------------------------------------------------------------
// Page copies: pool[dst[i]] = pool[src[i]], the pairs in the kernel's parameters (the host has
// checked them: in range, no page written twice or both read and written).
constexpr int COPY_PAIRS = 256;
struct CopyArgs {
    char* pool;
    long page_stride;           // bytes
    long page_bytes;            // multiple of 16
    int src[COPY_PAIRS], dst[COPY_PAIRS];
};

__global__ void __launch_bounds__(256) cache_copy_kernel(const __grid_constant__ CopyArgs a) {
    const uint4* s = reinterpret_cast<const uint4*>(a.pool + a.src[blockIdx.y] * a.page_stride);
    uint4* d = reinterpret_cast<uint4*>(a.pool + a.dst[blockIdx.y] * a.page_stride);
    const long n = a.page_bytes >> 4;
    for (long i = static_cast<long>(blockIdx.x) * blockDim.x + threadIdx.x; i < n;
         i += static_cast<long>(gridDim.x) * blockDim.x)
        d[i] = s[i];
}

// ---------------------------------------------------------------------------------------
// Accepted tokens: slot base + j of sequence b takes the K and V of slot base + keep[b][j], for
// j < n_keep[b], in every layer and head; new_base[b] = base[b] + n_keep[b]. keep is increasing, so
// keep[j] >= j: reading a run of rows before writing it, run after run, never reads a row that an
// earlier run has written.
struct KeepArgs {
    CachePlan plan;
    char* pool;
    long page_stride;           // bytes
    const int* keep;            // [B, A]
    long ld_keep;
    const int* n_keep;          // [B]
    int A;
    int* new_base;              // [B]
    int heads;                  // layers * 2 * KV head slabs in a page, page * D each
    int row_bytes;              // D * 2
};

// Whether sequence b's keep list is one the kernel may follow; the whole block calls it.
__device__ __forceinline__ bool keep_list_ok(const KeepArgs& a, int b) {
    const int n = a.n_keep[b];
    const int rows = a.plan.cu[b + 1] - a.plan.cu[b];
    const int base = a.plan.base[b];
    bool ok = n >= 0 && n <= a.A && base >= 0;
    if (ok)
        for (int j = threadIdx.x; j < n; j += blockDim.x) {
            const int i = a.keep[static_cast<long>(b) * a.ld_keep + j];
            const int before = j ? a.keep[static_cast<long>(b) * a.ld_keep + j - 1] : -1;
            int page, slot;
            ok = ok && i > before && i < rows && cache_slot(a.plan, b, static_cast<long>(base) + i, &page, &slot) &&
                 cache_slot(a.plan, b, static_cast<long>(base) + j, &page, &slot);
        }
    return __syncthreads_and(ok);
}

__global__ void __launch_bounds__(256) cache_keep_kernel(const KeepArgs a) {
    const int b = blockIdx.y, slab = blockIdx.x;
    const bool ok = keep_list_ok(a, b);
    const int base = a.plan.base[b], n = ok ? a.n_keep[b] : 0;
    if (slab == 0 && threadIdx.x == 0) {
        a.new_base[b] = base + n;
        if (!ok) record_bad_page();
    }
    const int vecs = a.row_bytes >> 4;                     // 16-byte pieces of a row
    const int rows = blockDim.x / vecs;                    // rows moved at once
    const int r = threadIdx.x / vecs, v = threadIdx.x % vecs;
    const long slab_off = static_cast<long>(slab) * a.row_bytes << a.plan.page_log2;
    for (int j0 = 0; j0 < n; j0 += rows) {
        const int j = j0 + r;
        uint4 x;
        bool move = false;
        if (j < n && r < rows) {
            const int i = a.keep[static_cast<long>(b) * a.ld_keep + j];
            int page, slot;
            move = i != j && cache_slot(a.plan, b, static_cast<long>(base) + i, &page, &slot);
            if (move)
                x = *reinterpret_cast<const uint4*>(a.pool + page * a.page_stride + slab_off +
                                                    static_cast<long>(slot) * a.row_bytes + v * 16);
        }
        __syncthreads();
        if (move) {
            int page, slot;
            if (cache_slot(a.plan, b, static_cast<long>(base) + j, &page, &slot))
                *reinterpret_cast<uint4*>(a.pool + page * a.page_stride + slab_off +
                                          static_cast<long>(slot) * a.row_bytes + v * 16) = x;
        }
        __syncthreads();
    }
}

}  // namespace mica
