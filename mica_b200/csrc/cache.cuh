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
// error word and touches no memory. A cu that passes the step's rows is recorded too (the rows that are
// there are served), and one that starts below zero or runs backwards: attention gives zeros then, append
// serves the rows that lie between both ends of a sequence. Rows that are no sequence's are padding.
#pragma once

#include "qk_rope.cuh"

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

// Records a cu that runs backwards, starts below zero or passes the rows; a whole warp calls it.
__device__ __forceinline__ void cache_check_cu(const CachePlan& p) {
    bool bad = p.cu[0] < 0 || p.cu[p.B] > p.N;
    for (int b = threadIdx.x & 31; b < p.B; b += 32) bad = bad || p.cu[b] > p.cu[b + 1];
    if (bad) record_bad_page();
}

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
    return lo < p.B && row >= p.cu[lo] && row < p.cu[lo + 1] ? lo : -1;
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

// Bound by the projection's bytes (read once, q and the pages written once). D / 8 lanes hold a
// head, 4 elements of its first half and their rotation partners of the second each (two 8-byte
// loads; with 16-byte ones the tables alone take the registers of half the warps), so a warp takes
// HP = 256 / D heads at a time and the sum of squares is a few shuffles.
// A row is one or more warps' (`split`: few rows are spread over the chip), each with every
// split-th set of HP heads; cos, sin and both norm weights stay in registers across them. The first
// loads of x are on their way while the row's place in the cache is looked up, and four sets are in
// flight. 8000 rows of 48 heads of 128 took 153 us with one warp a (row, head) and scalar loads, and take
// 55 us so, whatever the split (on fp32 pairs 65 to 88, with 16-byte loads 54 to 93: registers); rows in
// such numbers go through the ring below. Eight rows take 6 to 8 us, a launch.
// Keeps the words as they are in registers (their unpacked values, hoisted out of the loop, would take
// twice as many). Emits nothing.
__device__ __forceinline__ void keep_packed(uint2& q) { asm volatile("" : "+r"(q.x), "+r"(q.y)); }

template <int D>
__global__ void __launch_bounds__(256, 4) cache_append_kernel(const AppendArgs a, const int split) {
    constexpr int LPH = D / 8, HP = 32 / LPH;
    constexpr int AHEAD = 4;                     // sets in flight
    const long w = (static_cast<long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    const long row_l = w / split;
    if (row_l >= a.plan.N) return;
    const int row = static_cast<int>(row_l), part = static_cast<int>(w % split);
    const int heads = a.H + 2 * a.KV, sets = (heads + HP - 1) / HP;
    const int sub = lane / LPH, d = 4 * (lane % LPH);
    const __nv_bfloat16* x = a.qkv + static_cast<long>(row) * a.ld + d;
    uint2 lo[AHEAD], hi[AHEAD];
    const auto fetch = [&](int u, int set) {
        const int h = set * HP + sub;
        if (set < sets && h < heads) {
            lo[u] = *reinterpret_cast<const uint2*>(x + static_cast<long>(h) * D);
            hi[u] = *reinterpret_cast<const uint2*>(x + static_cast<long>(h) * D + D / 2);
        }
    };
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) fetch(u, part + u * split);

    // the row's slot and position
    long p = a.pos ? a.pos[row] : 0;
    const int b = cache_sequence_of(a.plan, row);
    bool ok = b >= 0;
    int page = 0, slot = 0;
    if (ok) {
        const int base = a.plan.base[b];
        const long index = static_cast<long>(base) + (row - a.plan.cu[b]);
        ok = base >= 0 && cache_slot(a.plan, b, index, &page, &slot);
        if (!a.pos) p = index;
        ok = ok && p >= 0 && p < a.n_pos;
        if (!ok && lane == 0) record_bad_page();
    }
    __nv_bfloat16* q = a.q_out + static_cast<long>(row) * a.ldq + d;
    if (!ok) {
        for (int set = part; set < sets; set += split) {
            const int h = set * HP + sub;
            if (h < a.H) {
                *reinterpret_cast<uint2*>(q + static_cast<long>(h) * D) = make_uint2(0u, 0u);
                *reinterpret_cast<uint2*>(q + static_cast<long>(h) * D + D / 2) = make_uint2(0u, 0u);
            }
        }
        if (w == 0) cache_check_cu(a.plan);
        return;
    }
    const auto pair = [&](const __nv_bfloat16* t, uint2& l, uint2& h) {
        l = __ldg(reinterpret_cast<const uint2*>(t + d));
        h = __ldg(reinterpret_cast<const uint2*>(t + d + D / 2));
    };
    uint2 cl, ch, sl, sh, ql, qh, kl, kh;
    pair(a.cos + p * D, cl, ch);
    pair(a.sin + p * D, sl, sh);
    pair(a.q_w, ql, qh);
    pair(a.k_w, kl, kh);
    const long slot_off = static_cast<long>(page) * a.page_stride + static_cast<long>(slot) * D + d;
    for (int set0 = part; set0 < sets; set0 += AHEAD * split) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int set = set0 + u * split;
            if (set >= sets) break;                          // uniform
            const int h = set * HP + sub;
            uint2 vl = lo[u], vh = hi[u];
            fetch(u, set + AHEAD * split);
            __nv_bfloat16* to = h < a.H ? q + static_cast<long>(h) * D
                                : (h < a.H + a.KV ? a.k_pages : a.v_pages) + slot_off +
                                      (static_cast<long>((h - a.H) % a.KV) << a.plan.page_log2) * D;
            float fl[4], fh[4], ss = 0.f;
            unpack4_bf16(vl, fl);
            unpack4_bf16(vh, fh);
#pragma unroll
            for (int e = 0; e < 4; ++e) ss = fmaf(fl[e], fl[e], fmaf(fh[e], fh[e], ss));
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (h < a.H + a.KV) {
                const float r = rsqrtf(ss * (1.f / D) + a.eps);
                keep_packed(cl); keep_packed(ch); keep_packed(sl); keep_packed(sh);
                keep_packed(ql); keep_packed(qh); keep_packed(kl); keep_packed(kh);
                float wl[4], wh[4], c0[4], c1[4], s0[4], s1[4];
                unpack4_bf16(h < a.H ? ql : kl, wl);
                unpack4_bf16(h < a.H ? qh : kh, wh);
                unpack4_bf16(cl, c0);
                unpack4_bf16(ch, c1);
                unpack4_bf16(sl, s0);
                unpack4_bf16(sh, s1);
                uint32_t ol[2], oh[2];
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    float y0[2], y1[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float a0 = fl[e + k] * r * wl[e + k], a1 = fh[e + k] * r * wh[e + k];
                        y0[k] = a0 * c0[e + k] - a1 * s0[e + k];
                        y1[k] = a1 * c1[e + k] + a0 * s1[e + k];
                    }
                    ol[e / 2] = pack_bf16(y0[0], y0[1]);
                    oh[e / 2] = pack_bf16(y1[0], y1[1]);
                }
                vl = make_uint2(ol[0], ol[1]);
                vh = make_uint2(oh[0], oh[1]);
            }
            if (h < heads) {
                *reinterpret_cast<uint2*>(to) = vl;
                *reinterpret_cast<uint2*>(to + D / 2) = vh;
            }
        }
    }
    if (w == 0) cache_check_cu(a.plan);          // one warp of the grid, its row sent
}

// The same for many rows: a CTA takes every grid-th row through a ring in shared memory. One warp looks
// up the places of 32 coming rows at once (a lane each) and keeps bulk copies of rows, cos and sin in
// flight; eight warps norm and turn q and k where they lie; one thread sends q, and each head's k and v,
// out by bulk copies. Nothing waits for a look-up or a load of its own row. 8000 rows of 48 heads of 128:
// 42 us, 5.0 TB/s read and written.
constexpr int APPEND_WARPS = 8, APPEND_STAGES = 8, APPEND_CTAS = 3;
constexpr long APPEND_SMEM = 70 << 10;      // of a CTA's ring
struct AppendStage {
    long off;                   // of the row's slot in a K or V page (elements, head 0)
    int row, ok;
};

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;"
                 ::"l"(reinterpret_cast<uint64_t>(dst)), "r"(smem_u32(src)), "r"(bytes) : "memory");
}

template <int D>
__global__ void __launch_bounds__(APPEND_WARPS * 32 + 64, APPEND_CTAS) cache_append_ring_kernel(const AppendArgs a, const int stages) {
    constexpr int LPH = D / 8, HP = 32 / LPH;
    extern __shared__ __align__(128) uint8_t append_ring[];
    __shared__ uint64_t full[APPEND_STAGES], done[APPEND_STAGES], empty[APPEND_STAGES];
    __shared__ AppendStage info[APPEND_STAGES];
    __shared__ uint32_t s_abort;
    volatile uint32_t* abort_flag = &s_abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t row_bytes = static_cast<uint32_t>(a.H + 2 * a.KV) * D * 2, stage_bytes = row_bytes + 4 * D;
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&done[i], APPEND_WARPS);
            mbar_init(&empty[i], 1);
        }
        s_abort = 0u;
        fence_mbar_init();
    }
    __syncthreads();
    const int rows = blockIdx.x < a.plan.N ? (a.plan.N - 1 - static_cast<int>(blockIdx.x)) / static_cast<int>(gridDim.x) + 1 : 0;
    if (warp == APPEND_WARPS) {
        // ---------------------------------- places and loads ----------------------------------
        int st = 0;
        uint32_t par = 1u;
        bool go = true;
        for (int i0 = 0; i0 < rows && go; i0 += 32) {
            // this lane's row of the next 32
            const int row = static_cast<int>(blockIdx.x) + (i0 + lane) * static_cast<int>(gridDim.x);
            long off = 0, p = 0;
            bool ok = false;
            if (i0 + lane < rows) {
                int lo = 0, n = a.plan.B;                       // ends cu[1..B] that are <= row
                while (n > 0) {
                    const int half = n >> 1;
                    if (a.plan.cu[lo + half + 1] <= row) { lo += half + 1; n -= half + 1; }
                    else n = half;
                }
                if (lo < a.plan.B && row >= a.plan.cu[lo] && row < a.plan.cu[lo + 1]) {
                    const int base = a.plan.base[lo];
                    const long index = static_cast<long>(base) + (row - a.plan.cu[lo]);
                    int page = 0, slot = 0;
                    ok = base >= 0 && cache_slot(a.plan, lo, index, &page, &slot);
                    p = a.pos ? a.pos[row] : index;
                    ok = ok && p >= 0 && p < a.n_pos;
                    off = static_cast<long>(page) * a.page_stride + static_cast<long>(slot) * D;
                    if (!ok) record_bad_page();
                }
            }
            const int n = min(32, rows - i0);
            for (int i = 0; i < n; ++i) {
                const long off_i = __shfl_sync(0xffffffffu, off, i), p_i = __shfl_sync(0xffffffffu, p, i);
                const int row_i = __shfl_sync(0xffffffffu, row, i);
                const bool ok_i = __shfl_sync(0xffffffffu, ok, i);
                bool w = true;
                if (lane == 0) {
                    w = mbar_wait(&empty[st], par, abort_flag, MICA_DEV_TIMEOUT_PRODUCER);
                    if (w) {
                        info[st].off = off_i;
                        info[st].row = row_i;
                        info[st].ok = ok_i;
                        uint8_t* to = append_ring + st * stage_bytes;
                        mbar_arrive_expect_tx(&full[st], ok_i ? stage_bytes : 0u);
                        if (ok_i) {
                            bulk_load(to, a.qkv + static_cast<long>(row_i) * a.ld, row_bytes, &full[st]);
                            bulk_load(to + row_bytes, a.cos + p_i * D, 2 * D, &full[st]);
                            bulk_load(to + row_bytes + 2 * D, a.sin + p_i * D, 2 * D, &full[st]);
                        }
                    }
                }
                go = __shfl_sync(0xffffffffu, w, 0);
                if (!go) break;
                if (++st == stages) { st = 0; par ^= 1u; }
            }
        }
        if (blockIdx.x == 0) cache_check_cu(a.plan);
        // copies in flight land before shared memory is released
        if (lane == 0)
            for (int i = max(0, rows - stages); i < rows; ++i)
                mbar_wait(&full[i % stages], (i / stages) & 1u, abort_flag, MICA_DEV_TIMEOUT_DRAIN);
        __syncwarp();
    } else if (warp == APPEND_WARPS + 1) {
        // ---------------------------------- stores ----------------------------------
        if (lane == 0) {
            int st = 0, before = -1;
            uint32_t par = 0u;
            for (int i = 0; i < rows; ++i) {
                if (!mbar_wait(&done[st], par, abort_flag, MICA_DEV_TIMEOUT_EPILOGUE)) break;
                const uint8_t* from = append_ring + st * stage_bytes;
                bulk_store(a.q_out + static_cast<long>(info[st].row) * a.ldq, from, a.H * D * 2);
                if (info[st].ok) {
                    from += a.H * D * 2;
                    const long off = info[st].off;
                    for (int h = 0; h < a.KV; ++h) {
                        const long at = off + (static_cast<long>(h) << a.plan.page_log2) * D;
                        bulk_store(a.k_pages + at, from + h * D * 2, D * 2);
                        bulk_store(a.v_pages + at, from + (a.KV + h) * D * 2, D * 2);
                    }
                }
                tma_store_commit();
                // the stage before has been read when all but this group are
                tma_store_wait_read<1>();
                if (before >= 0) mbar_arrive(&empty[before]);
                before = st;
                if (++st == stages) { st = 0; par ^= 1u; }
            }
            tma_store_wait_all<0>();
        }
        __syncwarp();
    } else {
        // ---------------------------------- norm and rotation ----------------------------------
        const int heads = a.H + a.KV, sub = lane / LPH, d = 4 * (lane % LPH);
        const auto pair = [&](const __nv_bfloat16* t, uint2& l, uint2& h) {
            l = *reinterpret_cast<const uint2*>(t + d);
            h = *reinterpret_cast<const uint2*>(t + d + D / 2);
        };
        uint2 ql, qh, kl, kh;
        pair(a.q_w, ql, qh);
        pair(a.k_w, kl, kh);
        int st = 0;
        uint32_t par = 0u;
        for (int i = 0; i < rows; ++i) {
            if (!__all_sync(0xffffffffu, mbar_wait(&full[st], par, abort_flag, MICA_DEV_TIMEOUT_EPILOGUE))) break;
            __nv_bfloat16* x = reinterpret_cast<__nv_bfloat16*>(append_ring + st * stage_bytes);
            if (info[st].ok) {
                uint2 c0, c1, n0, n1;
                pair(x + row_bytes / 2, c0, c1);
                pair(x + row_bytes / 2 + D, n0, n1);
                float cl[4], ch[4], sl[4], sh[4];
                unpack4_bf16(c0, cl);
                unpack4_bf16(c1, ch);
                unpack4_bf16(n0, sl);
                unpack4_bf16(n1, sh);
                for (int h0 = warp * HP; h0 < heads; h0 += APPEND_WARPS * HP) {
                    const int h = h0 + sub;
                    __nv_bfloat16* at = x + min(h, heads - 1) * D;
                    uint2 l, u;
                    pair(at, l, u);
                    float fl[4], fh[4], wl[4], wh[4], ss = 0.f;
                    unpack4_bf16(l, fl);
                    unpack4_bf16(u, fh);
#pragma unroll
                    for (int e = 0; e < 4; ++e) ss = fmaf(fl[e], fl[e], fmaf(fh[e], fh[e], ss));
#pragma unroll
                    for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                    const float r = rsqrtf(ss * (1.f / D) + a.eps);
                    unpack4_bf16(h < a.H ? ql : kl, wl);
                    unpack4_bf16(h < a.H ? qh : kh, wh);
                    float o0[4], o1[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float y0 = fl[e] * r * wl[e], y1 = fh[e] * r * wh[e];
                        o0[e] = y0 * cl[e] - y1 * sl[e];
                        o1[e] = y1 * ch[e] + y0 * sh[e];
                    }
                    if (h < heads) {
                        *reinterpret_cast<uint2*>(at + d) = make_uint2(pack_bf16(o0[0], o0[1]), pack_bf16(o0[2], o0[3]));
                        *reinterpret_cast<uint2*>(at + d + D / 2) = make_uint2(pack_bf16(o1[0], o1[1]), pack_bf16(o1[2], o1[3]));
                    }
                }
            } else {
                for (int e = threadIdx.x; e < a.H * D / 8; e += APPEND_WARPS * 32) reinterpret_cast<uint4*>(x)[e] = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async_smem();                       // the bulk stores read what was written here
            __syncwarp();
            if (lane == 0) mbar_arrive(&done[st]);
            if (++st == stages) { st = 0; par ^= 1u; }
        }
    }
    __syncthreads();
}

// ---------------------------------------------------------------------------------------
// Page copies: pool[dst[i]] = pool[src[i]], the pairs in the kernel's parameters (the host has
// checked them: in range, no page written twice or both read and written). Bound by memory: a block
// copies 32 KB, each thread's eight 16-byte loads under way before its first store; one load at a time
// reached 4.8 TB/s (read and written) over 61 pages of 9.4 MB, so it is 6.3.
constexpr int COPY_PAIRS = 256;
constexpr int COPY_AHEAD = 8;
struct CopyArgs {
    char* pool;
    long page_stride;           // bytes
    long page_bytes;            // multiple of 16
    int src[COPY_PAIRS], dst[COPY_PAIRS];
};

__global__ void __launch_bounds__(256) cache_copy_kernel(const __grid_constant__ CopyArgs a) {
    const uint4* s = reinterpret_cast<const uint4*>(a.pool + a.src[blockIdx.y] * a.page_stride);
    uint4* d = reinterpret_cast<uint4*>(a.pool + a.dst[blockIdx.y] * a.page_stride);
    const long n = a.page_bytes >> 4, i0 = static_cast<long>(blockIdx.x) * (256 * COPY_AHEAD) + threadIdx.x;
    uint4 x[COPY_AHEAD];
#pragma unroll
    for (int u = 0; u < COPY_AHEAD; ++u)
        if (i0 + u * 256 < n) x[u] = __ldcs(s + i0 + u * 256);
#pragma unroll
    for (int u = 0; u < COPY_AHEAD; ++u)
        if (i0 + u * 256 < n) __stcs(d + i0 + u * 256, x[u]);
}

// ---------------------------------------------------------------------------------------
// Accepted tokens: slot base + j of sequence b takes the K and V of slot base + keep[b][j], for
// j < n_keep[b], in every layer and head; new_base[b] = base[b] + n_keep[b]. keep is increasing, so
// keep[j] >= j: of rows taken in order, a later run never reads what an earlier one has written, and
// inside a run all are read before the first is written.
// A block checks the list once, leaves the places of the rows that move in shared memory, and takes
// `per_block` head slabs, KEEP_AHEAD at a time, 16-byte pieces side by side: 48 trees in 36 layers take
// 35 us (128 MB read and written), 63 with a block and its own check for each slab.
constexpr int KEEP_LIST = 256;
constexpr int KEEP_AHEAD = 8;
struct KeepArgs {
    CachePlan plan;
    char* pool;
    long page_stride;           // bytes
    const int* keep;            // [B, A]
    long ld_keep;
    const int* n_keep;          // [B]
    int A;
    int* new_base;              // [B]
    int slabs, per_block;       // layers * 2 * KV head slabs in a page, page * D each
    int row_bytes;              // D * 2
};

__device__ __forceinline__ void cache_keep_sequence(const KeepArgs& a, const int b) {
    __shared__ long s_src[KEEP_LIST], s_dst[KEEP_LIST];
    __shared__ int s_count[8], s_moves;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int base = a.plan.base[b], n = a.n_keep[b], rows = a.plan.cu[b + 1] - a.plan.cu[b];
    const int* list = a.keep + static_cast<long>(b) * a.ld_keep;
    // the list: increasing, below the row count, in pages of the pool
    bool ok = n >= 0 && n <= a.A && base >= 0;
    if (ok)
        for (int j = threadIdx.x; j < n; j += 256) {
            const int i = list[j], before = j ? list[j - 1] : -1;
            int page, slot;
            ok = ok && i > before && i < rows && cache_slot(a.plan, b, static_cast<long>(base) + i, &page, &slot) &&
                 cache_slot(a.plan, b, static_cast<long>(base) + j, &page, &slot);
        }
    ok = __syncthreads_and(ok);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        a.new_base[b] = base + (ok ? n : 0);
        if (!ok) record_bad_page();
    }
    if (!ok) return;
    const int slab0 = blockIdx.x * a.per_block, slab1 = min(a.slabs, slab0 + a.per_block);
    const long slab_bytes = static_cast<long>(a.row_bytes) << a.plan.page_log2;
    const int vecs = a.row_bytes >> 4, at_once = 256 / vecs;              // pieces of a row, rows of a run
    const int r = threadIdx.x / vecs, v = (threadIdx.x % vecs) * 16;
    for (int l0 = 0; l0 < n; l0 += KEEP_LIST) {
        // the rows of this part of the list that move, in order
        const int j = l0 + threadIdx.x, i = j < n ? list[j] : j;
        const uint32_t moves = __ballot_sync(0xffffffffu, i != j);
        if (lane == 0) s_count[warp] = __popc(moves);
        __syncthreads();
        int at = __popc(moves & ((1u << lane) - 1u));
        for (int w = 0; w < warp; ++w) at += s_count[w];
        if (i != j) {
            int page = 0, slot = 0;
            cache_slot(a.plan, b, static_cast<long>(base) + i, &page, &slot);
            s_src[at] = page * a.page_stride + static_cast<long>(slot) * a.row_bytes;
            cache_slot(a.plan, b, static_cast<long>(base) + j, &page, &slot);
            s_dst[at] = page * a.page_stride + static_cast<long>(slot) * a.row_bytes;
        }
        if (threadIdx.x == 255) s_moves = at + (i != j);
        __syncthreads();
        const int m = s_moves;
        for (int e0 = 0; e0 < m; e0 += at_once) {
            const bool mine = e0 + r < m;
            char* src = a.pool + (mine ? s_src[e0 + r] : 0) + v;
            char* dst = a.pool + (mine ? s_dst[e0 + r] : 0) + v;
            for (int s0 = slab0; s0 < slab1; s0 += KEEP_AHEAD) {
                uint4 x[KEEP_AHEAD];
#pragma unroll
                for (int u = 0; u < KEEP_AHEAD; ++u)
                    if (mine && s0 + u < slab1) x[u] = *reinterpret_cast<const uint4*>(src + (s0 + u) * slab_bytes);
                __syncthreads();
#pragma unroll
                for (int u = 0; u < KEEP_AHEAD; ++u)
                    if (mine && s0 + u < slab1) *reinterpret_cast<uint4*>(dst + (s0 + u) * slab_bytes) = x[u];
            }
        }
        __syncthreads();
    }
}

__global__ void __launch_bounds__(256) cache_keep_kernel(const KeepArgs a) {
    for (int b = blockIdx.y; b < a.plan.B; b += gridDim.y) cache_keep_sequence(a, b);
}

}  // namespace mica
