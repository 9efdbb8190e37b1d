// cache_attention.cuh -- grouped-query attention of a step's rows over a paged K/V cache, on
// tcgen05 (sm_100a).
//
//   o[i, h] = sum_s p_s V[s, h/G],  p = softmax over visible s of scale * q[i, h] . K[s, h/G]
//
// Row i of sequence b sees every committed token (s < base[b]) and node j of its own step
// (s = base[b] + j) when bit j of mask[row] is set, or, without a mask, when j <= i. A row that
// sees nothing gives zero.
//
// What bounds it: for a few rows the K and V bytes (each is read once: 4 D bytes a key and K/V
// head), for T rows of G heads each above about 250 the tensor cores. So the G heads of a K/V
// head share its tiles (row r of a 128-row tile is head r % G of node r / G, which a 3-D TMA box of
// q lays down as it is), and the key axis is cut wherever the SMs need it:
//
// Work. A unit is (sequence, K/V head, block of NT * npt nodes); its key tiles of 128 follow one
// another, units in order, in one line (where each unit has some places more for what it costs by
// itself, and tiles that are shared by two row tiles count for more). Each of the CTAs (one per SM)
// takes an equal run of that line, whatever the lengths: it starts and may end inside a unit. A unit
// that one CTA has whole is written out; of a divided one each CTA leaves its unnormalised rows, maxima
// and sums in its own place of the workspace (a CTA has at most two such: its first and its last), and
// cache_attention_join adds them up in the order of the CTAs. No atomics: the same bits every time.
// The lengths are read on the device, so a captured graph serves any.
//
// Warps: 0 loads Q and K tiles, 2 V tiles, by TMA page by page: one box per page and 64 columns, one
// lane each, the page numbers fetched a tile ahead (a box takes the warp about 90 cycles, so that with
// pages of 16 one warp for both was as slow as memory); 1 issues the MMAs (S = Q K^T both from
// shared memory, O += P V with P in tensor memory); the others softmax, one row a thread, as in
// attention.cuh. NT = 1: S and P have two buffers each, so scores, softmax and P.V of three
// consecutive tiles overlap; Q has two, so the next unit's loads run under this one's end. Up to 16 rows
// (8 of D = 128) lie in the row tile four times, once in each warp's quarter of tensor memory, and each warp
// takes 32 keys of a tile for them in place of 128, with its own maximum, sum and accumulator (its weights
// are zero for the others' keys); a unit's end adds the four up, which costs more than it gains at more
// rows (64 sequences of 300 to 4000 keys, 32 heads over 8 of 64: 90 -> 78 us with 16 rows, 89 -> 93 with 32). NT = 2:
// two row tiles share every K and V tile (attention.cuh's schedule).
// P is rounded to bf16 for the tensor core (V's type): each weight is off by a half step, 2^-8 of it at
// most, and these errors are independent, so the result is off by about as much as its own rounding to
// bf16; the row sum is taken in fp32 before that.
//
// Keys that a row does not see get score -inf. A weight of zero still meets its V row in the MMA, and
// 0 * NaN is not zero: in the tiles that some row of the unit does not see all of (they hold nodes of
// the step, or the end of the keys), V rows behind the end are zeroed in shared memory, and an infinite
// or NaN element of a node's V is replaced by zero and added to the accumulators of the rows that see
// it, no others.
//
// Measured (32 heads over 8, D = 128, cold L2, in a graph): 13 and 15 tokens over 70761 and 87495 keys 131 us (117
// warm), the key tiles among them at the memory's 6.5 TB/s (1.5 us a tile and SM); 16 trees of up to 64 nodes over up
// to 9000 keys 90 us, a tile of two row tiles 1.7 us (softmax: 2100 cycles of it the scores' way through the
// exponential, 1100 waits, packing and stores); 700 nodes over 20000 keys 212 us, 1.08 PFLOP/s (calls back to back,
// under the power cap, 241 us, 0.95); 8192 causal rows 530 us, 1.04 PFLOP/s; one token over up to 700 keys 18 us
// with its launch and the join. D = 64: 8 tokens over eight contexts of 8000, 24 heads over 8, 56 us against 20 for
// the bytes: one softmax warpgroup takes 1.3 us a tile, whose bytes take half of D = 128's time.
#pragma once

#include "attention.cuh"
#include "cache.cuh"

namespace mica {

struct CacheAttnArgs {
    CachePlan plan;
    const __nv_bfloat16* v_pages;
    long page_stride;           // elements
    const unsigned long long* mask;   // [N, ld_mask] or nullptr (causal)
    long ld_mask;
    int words;                  // 64-bit words of a row's mask
    __nv_bfloat16* out;         // [N, ldo]
    long ldo;
    int KV, G;                  // K/V heads, query heads of each
    int npt;                    // nodes of a row tile: npt * G <= 128
    bool quarters;              // the rows lie in the row tile four times (npt * G * D <= 1024; NT 1)
    int ctas;                   // CTAs of the grid
    float scale_log2;           // scale * log2(e)
    float* ws;                  // partials: [ctas][2] places
    int4* cuts;                 // [ctas][2] the unit a CTA starts inside, for the CTA that is the first to (w -1: cu is
                                // out of order)
};

// A place of the workspace: rows of O as [NT][D / 4][128] float4 (a warp's rows side by side), then
// (max, sum) [NT][128].
template <int D, int NT>
__host__ __device__ constexpr long cache_attn_place_floats() { return NT * 128l * (D + 2); }

// ---- the line of tiles ----------------------------------------------------------------
struct CacheSeq {
    int row0, T, base, keys;    // first row, rows, committed tokens, keys (0: not usable)
};
__device__ __forceinline__ CacheSeq cache_seq(const CachePlan& p, int b) {
    CacheSeq s;
    s.row0 = min(max(p.cu[b], 0), p.N);
    s.T = max(min(p.cu[b + 1], p.N) - s.row0, 0);
    s.base = p.base[b];
    const long keys = static_cast<long>(s.base) + s.T;
    s.keys = s.base < 0 || keys > (static_cast<long>(p.P) << p.page_log2) ? 0 : static_cast<int>(keys);
    return s;
}
// Key tiles of the row block `rb` (R nodes each): all keys under a mask, else up to its last node.
// At least one, so that every row is written.
__device__ __forceinline__ int cache_unit_tiles(const CacheSeq& s, int rb, int R, bool causal) {
    int keys = s.keys;
    if (causal && keys) keys = s.base + min(s.T, (rb + 1) * R);
    return max(1, (keys + 127) >> 7);
}
__device__ __forceinline__ int cache_row_blocks(const CacheSeq& s, int R) { return (s.T + R - 1) / R; }
// What a unit counts in the line: its tiles and UNIT more (its rows' way out, nothing in flight), times a
// weight for a tile, 4 with two row tiles and 3 where its nodes fill only one of the two.
template <int NT>
struct CacheCost {
    static constexpr int UNIT = 2;
    static constexpr int TILE = NT == 1 ? 1 : 4;
    __device__ __forceinline__ static int weight(const CacheSeq& s, int rb, int R) {
        return NT == 1 ? 1 : s.T - rb * R <= R / 2 ? 3 : 4;
    }
    __device__ __forceinline__ static long seq(const CacheSeq& s, int R, bool causal) {      // of one K/V head
        const int n = cache_row_blocks(s, R);
        if (n == 0) return 0;
        long t = static_cast<long>(cache_unit_tiles(s, n - 1, R, causal) + UNIT) * weight(s, n - 1, R);
        if (!causal) return t + static_cast<long>(n - 1) * (cache_unit_tiles(s, 0, R, false) + UNIT) * TILE;
        for (int rb = 0; rb + 1 < n; ++rb) t += static_cast<long>(cache_unit_tiles(s, rb, R, true) + UNIT) * TILE;
        return t;
    }
};

struct CachePlace {             // a place of the line: the off-th of sequence b
    long total;
    long off;
    int b;
};
// The line's length and the sequence that holds place `first(total)`; every thread of the block calls it.
template <int NT, typename F>
__device__ __forceinline__ CachePlace cache_locate(const CachePlan& p, int KV, int R, bool causal, F first) {
    __shared__ long s_warp[32];
    __shared__ long s_off;
    __shared__ int s_b;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (blockDim.x + 31) >> 5;
    const auto scan = [&](long v, long& all) {       // inclusive over the block
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        __syncthreads();
        if (lane == 31) s_warp[warp] = v;
        __syncthreads();
        all = 0;
        for (int i = 0; i < warps; ++i) {
            if (i < warp) v += s_warp[i];
            all += s_warp[i];
        }
        return v;
    };
    const auto tiles = [&](int b) { return b < p.B ? KV * CacheCost<NT>::seq(cache_seq(p, b), R, causal) : 0l; };
    if (p.B <= 32) {                                 // every warp by itself
        const long n = tiles(lane);
        long end = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long u = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end += u;
        }
        const long total = __shfl_sync(0xffffffffu, end, 31), t = first(total);
        const uint32_t here = __ballot_sync(0xffffffffu, t >= end - n && t < end);
        const int b = __ffs(here) - 1;
        return CachePlace{total, t - __shfl_sync(0xffffffffu, end - n, max(b, 0)), b};
    }
    const long mine = tiles(threadIdx.x);
    long total = 0;
    if (threadIdx.x == 0) { s_b = -1; s_off = 0; }
    if (p.B <= static_cast<int>(blockDim.x)) {
        const long end = scan(mine, total), t = first(total);
        if (t >= end - mine && t < end) {
            s_b = threadIdx.x;
            s_off = t - (end - mine);
        }
        __syncthreads();
        return CachePlace{total, s_off, s_b};
    }
    long sum = mine;
    for (int b = threadIdx.x + blockDim.x; b < p.B; b += blockDim.x) sum += tiles(b);
    scan(sum, total);
    const long t = first(total);
    long before = 0;
    for (int b0 = 0; b0 < p.B; b0 += blockDim.x) {
        const long n = b0 == 0 ? mine : tiles(b0 + threadIdx.x);
        long all = 0;
        const long end = before + scan(n, all);      // its barriers order s_b's first write
        if (t >= end - n && t < end) {
            s_b = b0 + threadIdx.x;
            s_off = t - (end - n);
        }
        before += all;
        if (before > t) break;
    }
    __syncthreads();
    return CachePlace{total, s_off, s_b};
}

// The runs of the CTAs: total / used places each, the first total % used one more. Fewer CTAs are used
// when there are fewer tiles, so that a run has a tile's places at least.
struct CacheShare {
    long each;
    int rest, used;
    __device__ __forceinline__ CacheShare(long total, int ctas, int tile) {
        const long most = total / tile;
        used = static_cast<int>(most < ctas ? most : ctas);
        if (total <= 0x7fffffffl) {
            const unsigned n = static_cast<unsigned>(total), d = max(used, 1);
            each = n / d;
            rest = static_cast<int>(n - static_cast<unsigned>(each) * d);
        } else {
            each = total / max(used, 1);
            rest = static_cast<int>(total - each * used);
        }
    }
    __device__ __forceinline__ long at(int c) const { return each * c + min(c, rest); }
};

// The units of a CTA's run, one after another: those of which it has tiles. A tile is the run's that holds
// the first of its places; a unit's first UNIT tiles' places are nobody's.
template <int NT>
struct CacheWalk {
    using Cost = CacheCost<NT>;
    CacheSeq s;
    int b, kvh, rb;             // unit
    int nk, j0, j1;             // its tiles, and the CTA's [j0, j1) of them
    int w;                      // places of a tile
    long left;                  // places of the run from the unit's first on
    int R;
    bool causal;

    __device__ __forceinline__ long unit_places() const { return static_cast<long>(nk + Cost::UNIT) * w; }
    __device__ __forceinline__ int tiles_before(long places) const {       // of those places of the unit
        if (places >= unit_places()) return nk;
        return max(0, static_cast<int>((static_cast<unsigned>(places) + w - 1) / static_cast<unsigned>(w)) - Cost::UNIT);
    }
    __device__ __forceinline__ void unit() {
        nk = cache_unit_tiles(s, rb, R, causal);
        w = Cost::weight(s, rb, R);
    }
    // off: the run's first place in sequence b_; false: it has no tile
    __device__ __forceinline__ bool start(const CachePlan& p, int KV, int R_, bool causal_, int b_, long off, long n) {
        R = R_; causal = causal_; b = b_;
        s = cache_seq(p, b);
        const long per = Cost::seq(s, R, causal);
        kvh = off <= 0x7fffffffl && per <= 0x7fffffffl ? static_cast<int>(static_cast<unsigned>(off) / static_cast<unsigned>(per))
                                                       : static_cast<int>(off / per);
        off -= kvh * per;
        rb = 0;
        for (unit(); off >= unit_places(); unit()) { off -= unit_places(); ++rb; }
        left = n + off;
        j0 = tiles_before(off);
        if (j0 == nk) return next(p, KV);                   // behind the first place of its last tile
        j1 = tiles_before(left);
        return j1 > j0;
    }
    __device__ __forceinline__ bool next(const CachePlan& p, int KV) {
        left -= unit_places();
        if (left <= 0) return false;
        if (++rb >= cache_row_blocks(s, R)) {
            rb = 0;
            if (++kvh >= KV) {
                kvh = 0;
                do {
                    if (++b >= p.B) return false;
                    s = cache_seq(p, b);
                } while (s.T == 0);
            }
        }
        unit();
        j0 = 0;
        j1 = tiles_before(left);
        return j1 > 0;
    }
    __device__ __forceinline__ bool whole() const { return j0 == 0 && j1 == nk; }
};

// What a role needs of the unit it is at: the K warp walks the run and leaves it here, four units deep. A
// place is taken again once every warp that reads it (MMA, V, softmax) has said that it is done with the unit
// before: row tile 1's warps pass over units that have no rows for them, and nothing else holds the K warp,
// or the parity of unit_full, to their pace.
struct CacheUnit {
    int b, kvh, row0, node0, nodes;     // row0: global row of its first node (node0 of its sequence)
    int base, keys, j0, j1;
    int special;                        // the first tile that some row does not see all of, or that ends the keys
    int flags;                          // 1: the run's last unit, 2: all of the unit's tiles, 4: the run's first unit,
                                        // 8: its nodes fill one row tile at most
};
constexpr int CACHE_UNITS = 4;

template <int D, int NT>
struct CacheAttnShape {
    static constexpr int HALVES = D / 64;
    static constexpr int TILE = 128 * D * 2;
    static constexpr int QBUF = NT == 1 ? 2 : 1;
    static constexpr int KST = D == 128 ? 3 : 6;
    static constexpr int VST = D == 128 ? 2 : 5;
    static constexpr int THREADS = 128 + 128 * NT;
    static constexpr int BARS = D == 128 ? 576 : 672;                     // barriers and units
    static constexpr int STATS = NT == 1 ? 128 * 8 : 0;                  // the copies' (max, sum)
    static constexpr int SMEM = 1024 + TILE * (QBUF * NT + KST + VST) + BARS + STATS;
    static_assert((4 + 2 * KST + 2 * VST + 8 + 1 + 2 * CACHE_UNITS + 2) * 8 + 8 + 64 + CACHE_UNITS * sizeof(CacheUnit) <= BARS, "BARS");
};

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

// 128 bits of a row's mask words from bit `off` (which may be negative) on, bits outside them zero.
__device__ __forceinline__ void mask_bits(const unsigned long long* m, int words, int off, uint32_t (&out)[4]) {
    const int w = off >> 6, sh = off & 63;                     // floor
    unsigned long long v[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) v[i] = w + i >= 0 && w + i < words ? m[w + i] : 0ull;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const unsigned long long x = sh ? v[i] >> sh | v[i + 1] << (64 - sh) : v[i];
        out[2 * i] = static_cast<uint32_t>(x);
        out[2 * i + 1] = static_cast<uint32_t>(x >> 32);
    }
}
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// Rows first .. end - 1 of the output stay as they are, all others become zero: by `threads` of each of the blocks.
__device__ __forceinline__ void cache_zero_rows(const CacheAttnArgs& args, int D, int first, int end, long block, long blocks,
                                                int thread, int threads) {
    const int N = args.plan.N, vecs = args.KV * args.G * D / 8;
    for (long i_row = block; i_row < N - (end - first); i_row += blocks) {
        const long row = i_row < first ? i_row : i_row - first + end;
        for (int i = thread; i < vecs; i += threads)
            *reinterpret_cast<uint4*>(args.out + row * args.ldo + i * 8) = make_uint4(0u, 0u, 0u, 0u);
    }
}
// Rows before the first sequence and behind the last become zero.
__device__ __forceinline__ void cache_zero_padding(const CacheAttnArgs& args, int D, int thread, int threads) {
    const int N = args.plan.N, first = min(max(args.plan.cu[0], 0), N);
    cache_zero_rows(args, D, first, max(first, min(args.plan.cu[args.plan.B], N)), blockIdx.x, gridDim.x, thread, threads);
}
// Looks the row offsets over, by one warp; false when they run backwards or start below zero: two sequences may
// claim a row then, and the join makes all rows zero.
__device__ __noinline__ bool cache_ordered(const CachePlan& p) {
    bool bad = false;
    for (int b = threadIdx.x & 31; b < p.B; b += 32) bad = bad || p.cu[b] < 0 || p.cu[b] > p.cu[b + 1];
    const bool ordered = !__any_sync(0xffffffffu, bad);
    if (blockIdx.x == 0 && (threadIdx.x & 31) == 0 && (!ordered || p.cu[p.B] > p.N)) record_bad_page();
    return ordered;
}

// The keys k0 .. k0 + 127 that node `node` of unit u's sequence sees (row: its row of the step), one bit
// each; in the tiles that hold nodes of the step or the end of the keys.
__device__ __forceinline__ void cache_visible(const CacheAttnArgs& args, const volatile CacheUnit& u, int x, int node_r,
                                              int k0, uint32_t (&vis)[4]) {
    const int base = u.base, keys = u.keys, node = x * args.npt + node_r;
    const bool live = node_r < args.npt && node < u.nodes && keys > 0;
    const bool causal = args.mask == nullptr;
    const int end = causal ? min(keys, base + u.node0 + node + 1) : keys;
    uint32_t bits[4] = {~0u, ~0u, ~0u, ~0u};
    if (!causal && live)
        mask_bits(args.mask + static_cast<long>(u.row0 + node) * args.ld_mask, args.words, k0 - base, bits);
#pragma unroll
    for (int w = 0; w < 4; ++w)
        vis[w] = live ? low_bits(end - k0 - 32 * w) & (low_bits(base - k0 - 32 * w) | bits[w]) : 0u;
}
// Row r (key k0 + r) of columns 64 h0 .. of a V tile in shared memory, made safe for weights of zero: rows
// behind the keys become zero, infinities and NaN of the step's own rows too. Returns whether there were any.
__device__ __forceinline__ bool cache_fix_v(uint8_t* tile, int r, int h0, int h1, bool behind) {
    bool odd = false;
    for (int h = h0; h < h1; ++h) {
        uint4* vr = reinterpret_cast<uint4*>(tile + h * ATT_HALF_BYTES + r * 128);
        if (behind) {
#pragma unroll
            for (int e = 0; e < 8; ++e) vr[e ^ (r & 7)] = make_uint4(0u, 0u, 0u, 0u);
            continue;
        }
        // 0 * v is zero for finite v only
        __nv_bfloat162 any = bf2(0u);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint4 v = vr[e ^ (r & 7)];
            any = __hfma2(bf2(v.x), bf2(0u), any);
            any = __hfma2(bf2(v.y), bf2(0u), any);
            any = __hfma2(bf2(v.z), bf2(0u), any);
            any = __hfma2(bf2(v.w), bf2(0u), any);
        }
        if (bits2(any) & 0x7fff7fffu) {
            odd = true;
            uint32_t* u = reinterpret_cast<uint32_t*>(vr);
            for (int e = 0; e < 32; ++e) {
                if ((u[e] & 0x7f800000u) == 0x7f800000u) u[e] &= 0x0000ffffu;
                if ((u[e] & 0x00007f80u) == 0x00007f80u) u[e] &= 0xffff0000u;
            }
        }
    }
    return odd;
}

// Whether the fixes-th special tile has odd values.
template <int NT>
__device__ __forceinline__ bool cache_any_odd(const volatile uint32_t* odd_v, int fixes) {
    const volatile uint32_t* odd = odd_v + (fixes & 1) * 4 * NT;
    uint32_t some = 0u;
#pragma unroll
    for (int i = 0; i < 4 * NT; ++i) some |= odd[i];
    return some != 0u;
}

// A tile of V that holds nodes of the step or the end of the keys, made safe by the softmax warps: each waits
// for it, takes its rows (two row tiles half of the columns each), leaves in `odd` which had odd values, and
// arrives on v_fixed. (`odd` is one of two sets: all warps pass v_fixed of a special tile before one writes the
// next but one.)
template <int D, int NT>
__device__ __noinline__ bool cache_safe_v(uint8_t* tile, uint64_t* full, uint32_t parity, uint64_t* v_fixed, uint32_t* odd,
                                          const volatile CacheUnit& u, int k0, int x, volatile uint32_t* abort_flag) {
    if (!__all_sync(0xffffffffu, mbar_wait(full, parity, abort_flag, MICA_DEV_TIMEOUT_EPILOGUE))) return false;
    constexpr int HALVES = D / 64;
    const int lane = threadIdx.x & 31, q4 = (threadIdx.x >> 5) & 3, r = q4 * 32 + lane, key = k0 + r;
    const bool alone = NT == 1 || (u.flags & 8);
    bool any = false;
    if (key >= u.base || key >= u.keys)
        any = cache_fix_v(tile, r, alone ? 0 : x, alone ? HALVES : min(x + 1, HALVES), key >= u.keys);
    const uint32_t found = __ballot_sync(0xffffffffu, any);
    fence_proxy_async_smem();
    if (lane == 0) {
        odd[x * 4 + q4] = found;
        if (NT == 2 && alone) odd[4 + q4] = 0u;
    }
    __syncwarp();
    if (lane == 0) {
        mbar_arrive(v_fixed);
        if (NT == 2 && alone) mbar_arrive(v_fixed);          // for row tile 1's warp
    }
    return true;
}

// Copies of the rows meet the keys of one another with weights of zero, and 0 * infinity is NaN: a sum that is
// not finite is set to what the infinities and NaN among the V that its row sees in this CTA's tiles make of it.
// Three bits for each of 4 columns from `col`: NaN, infinity, -infinity. The whole warp calls it; mend: this
// thread's row and columns are asked for.
template <int D>
__device__ __noinline__ uint32_t cache_odd_kinds(const CacheAttnArgs& args, const volatile CacheUnit& u, int node_r, int col,
                                                 bool mend) {
    const CachePlan& plan = args.plan;
    const int lane = threadIdx.x & 31, b = u.b, special = u.special;
    const auto kinds = [&](int key, int c0) {
        int page = 0, slot = 0;
        if (!cache_slot(plan, b, key, &page, &slot)) return 0u;
        const uint16_t* v = reinterpret_cast<const uint16_t*>(args.v_pages) + page * args.page_stride +
                            ((static_cast<long>(u.kvh) << plan.page_log2) + slot) * D + c0;
        uint32_t k = 0u;
        for (int e = 0; e < 4; ++e) {
            const uint32_t bits = v[e];
            if ((bits & 0x7f80u) == 0x7f80u) k |= (bits & 0x7fu ? 1u : bits & 0x8000u ? 4u : 2u) << (3 * e);
        }
        return k;
    };
    // the tiles whose keys all rows see, for one set of columns after the other
    uint32_t mine = 0u;
    for (uint32_t todo = __ballot_sync(0xffffffffu, mend); todo;) {
        const int c0 = __shfl_sync(0xffffffffu, col, __ffs(todo) - 1);
        uint32_t k = 0u;
        for (int key = u.j0 * 128 + lane; key < min(u.j1, special) * 128; key += 32) k |= kinds(key, c0);
        k = __reduce_or_sync(0xffffffffu, k);
        if (col == c0) mine = k;
        todo &= ~__ballot_sync(0xffffffffu, col == c0);
    }
    for (int j = max(u.j0, special); mend && j < u.j1; ++j) {
        uint32_t vis[4];
        cache_visible(args, u, 0, node_r, j * 128, vis);
        for (int i = 0; i < 128; ++i) {
            const uint32_t seen = i < 64 ? (i < 32 ? vis[0] : vis[1]) : (i < 96 ? vis[2] : vis[3]);
            if (seen >> (i & 31) & 1u) mine |= kinds(j * 128 + i, col);
        }
    }
    return mend ? mine : 0u;
}

// A row's weights are 2^fma(s, c, -m), for scores s as they come from the MMA, c = scale * log2(e) and the running
// maximum m = fl(max c), whose rounding is a factor of all of them and cancels. Beyond |m| = 2^30 that rounding may
// take them out of fp32's range, and scores that differ at all differ by 64 or more, so only those equal to the
// largest count: the power of two above c stands in for c there, with which both products are exact. m stays in
// order across the limit, so sums with different maxima are brought together by 2^(m - m') either way. Nothing
// seen yet: CACHE_NOTHING. (Scores have to stay within fp32's range when they are multiplied by that.)
constexpr float CACHE_FAR = 1073741824.f, CACHE_NOTHING = -3e38f;

template <int D, int NT>
__global__ void __launch_bounds__(CacheAttnShape<D, NT>::THREADS, 1)
cache_attention_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                       const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ CacheAttnArgs args) {
    using S = CacheAttnShape<D, NT>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const CachePlan& plan = args.plan;
    const bool causal = args.mask == nullptr;
    const int R = NT * args.npt;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");    // the join kernel may take its place
    const int cta = blockIdx.x;
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmap_q);
        tma_prefetch_desc(&tmap_k);
        tma_prefetch_desc(&tmap_v);
    }
    // this CTA's run of tiles
    using Cost = CacheCost<NT>;
    const CachePlace place = cache_locate<NT>(plan, args.KV, R, causal,
                                              [&](long total) { return CacheShare(total, args.ctas, Cost::TILE).at(cta); });
    const CacheShare share(place.total, args.ctas, Cost::TILE);
    CacheWalk<NT> wk;
    if (cta >= share.used || place.b < 0 ||
        !wk.start(plan, args.KV, R, causal, place.b, place.off, share.at(cta + 1) - share.at(cta))) {
        if (warp == 3) {
            const bool ordered = cache_ordered(plan);
            if (lane == 0) args.cuts[2 * cta] = make_int4(0, 0, 0, ordered ? 0 : -1);
        }
        cache_zero_padding(args, D, threadIdx.x, blockDim.x);
        return;
    }

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* sq = smem;
    uint8_t* sk = sq + S::QBUF * NT * S::TILE;
    uint8_t* sv = sk + S::KST * S::TILE;
    uint64_t* q_full = reinterpret_cast<uint64_t*>(sv + S::VST * S::TILE);   // [QBUF]
    uint64_t* q_empty = q_full + 2;
    uint64_t* k_full = q_empty + 2;
    uint64_t* k_empty = k_full + S::KST;
    uint64_t* v_full = k_empty + S::KST;
    uint64_t* v_empty = v_full + S::VST;
    uint64_t* s_full = v_empty + S::VST;       // [2] scores written: by buffer (NT 1) or row tile (NT 2)
    uint64_t* s_free = s_full + 2;             // [2] scores read
    uint64_t* p_full = s_free + 2;             // [2] P written
    uint64_t* pv_done = p_full + 2;            // [2] P.V finished
    uint64_t* v_fixed = pv_done + 2;           // V of a special tile made safe (all softmax warps)
    uint64_t* unit_full = v_fixed + 1;         // [CACHE_UNITS]
    uint64_t* unit_empty = unit_full + CACHE_UNITS;   // [CACHE_UNITS] read by the MMA, V and softmax warps
    uint64_t* drain = unit_empty + CACHE_UNITS;
    uint64_t* exchange = drain + 1;            // the copies' rows of a unit are all there
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(exchange + 1);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    uint32_t* odd_v = tmem_slot + 2;           // [2][NT][4] keys of a special tile whose V row holds infinities or NaN
    volatile CacheUnit* units = reinterpret_cast<volatile CacheUnit*>(odd_v + 16);
    float2* stats = reinterpret_cast<float2*>(sv + S::VST * S::TILE + S::BARS);
    const bool quarters = NT == 1 && args.quarters;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], quarters ? 5 : 1);         // the softmax warps add the copies up in it
            mbar_init(&s_full[i], 1);
            mbar_init(&s_free[i], 4);
            mbar_init(&p_full[i], 4);
            mbar_init(&pv_done[i], 1);
        }
        for (int i = 0; i < S::KST; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); }
        for (int i = 0; i < S::VST; ++i) { mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1); }
        mbar_init(v_fixed, 4 * NT);
        for (int i = 0; i < CACHE_UNITS; ++i) {
            mbar_init(&unit_full[i], 1);
            mbar_init(&unit_empty[i], 2 + 4 * NT);
        }
        mbar_init(drain, 1);
        mbar_init(exchange, 4);
        *abort_flag = 0u;
        fence_mbar_init();
    }
    if (warp == 1) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // tensor memory columns: NT 1: S [0,128) [128,256) P [256,320) [320,384) O [384,512);
    //                        NT 2: S [0,128) P [128,192) [192,256) O [256,384) [384,512)
    const auto col_s = [](int i) { return NT == 1 ? i * 128 : 0; };
    const auto col_p = [](int i) { return (NT == 1 ? 256 : 128) + i * 64; };
    const auto col_o = [](int x) { return NT == 1 ? 384 : 256 + x * 128; };

    if (warp == 0 || warp == 2) {
        // ---------------------------------- producers ---------------------------------
        const bool is_k = warp == 0;
        const int stages = is_k ? S::KST : S::VST;
        uint64_t* const full = is_k ? k_full : v_full;
        uint64_t* const empty = is_k ? k_empty : v_empty;
        uint8_t* const ring = is_k ? sk : sv;
        const CUtensorMap* const map = is_k ? &tmap_k : &tmap_v;
        const int ppt = 128 >> plan.page_log2;             // pages of a key tile
        const int boxes = ppt * S::HALVES;                 // <= 16, lane i: page i / HALVES, columns 64 (i % HALVES)
        const int my_page = lane / S::HALVES, my_half = lane % S::HALVES;
        const uint32_t box_bytes = 128u << plan.page_log2;
        const int page = 1 << plan.page_log2;
        bool ok = true, last = false;
        int t = 0, st = 0, unit = 0;                       // tiles, ring stage, units
        uint32_t par = 1u;                                 // of the stage's `empty`
        for (; !last && ok; ++unit) {
            const int slot = unit % CACHE_UNITS;
            if (is_k) {
                const int qb = S::QBUF == 2 ? unit & 1 : 0;
                bool w = true;
                if (lane == 0) {
                    w = mbar_wait(&q_empty[qb], static_cast<uint32_t>(unit / S::QBUF & 1) ^ 1u, abort_flag,
                                  MICA_DEV_TIMEOUT_PRODUCER) &&
                        mbar_wait(&unit_empty[slot], static_cast<uint32_t>(unit / CACHE_UNITS & 1) ^ 1u, abort_flag,
                                  MICA_DEV_TIMEOUT_PRODUCER);
                    if (w) {
                        const int copies = quarters ? 4 : 1;
                        if (wk.s.keys == 0) record_bad_page();
                        const int node0 = wk.rb * R;
                        mbar_arrive_expect_tx(&q_full[qb], NT * copies * S::HALVES * 128u * args.npt * args.G);
                        for (int x = 0; x < NT * copies; ++x)        // one of the two is 1
                            for (int h = 0; h < S::HALVES; ++h)
                                tma_load_3d(NT == 1 ? sq + qb * S::TILE + h * ATT_HALF_BYTES + x * (ATT_HALF_BYTES / copies)
                                                    : sq + x * S::TILE + h * ATT_HALF_BYTES, &tmap_q, &q_full[qb], h * 64,
                                            wk.kvh * args.G, wk.s.row0 + node0 + (NT == 1 ? 0 : x) * args.npt);
                        volatile CacheUnit& u = units[slot];
                        u.b = wk.b; u.kvh = wk.kvh; u.row0 = wk.s.row0 + node0; u.node0 = node0; u.nodes = min(R, wk.s.T - node0);
                        u.base = wk.s.base; u.keys = wk.s.keys; u.j0 = wk.j0; u.j1 = wk.j1;
                        // every row sees the committed tokens, and without a mask what the first row sees
                        u.special = wk.s.keys ? min(wk.s.keys, wk.s.base + (causal ? node0 + 1 : 0)) >> 7 : 0;
                        const int all = wk.whole() ? 2 : 0;
                        u.flags = (wk.next(plan, args.KV) ? 0 : 1) | all | (unit == 0 ? 4 : 0) | (u.nodes <= args.npt ? 8 : 0);
                        mbar_arrive(&unit_full[slot]);
                    }
                }
                ok = __shfl_sync(0xffffffffu, w, 0);
                __syncwarp();
            } else {
                ok = __all_sync(0xffffffffu, mbar_wait(&unit_full[slot], unit / CACHE_UNITS & 1, abort_flag,
                                                       MICA_DEV_TIMEOUT_PRODUCER));
            }
            if (!ok) break;
            const volatile CacheUnit& u = units[slot];
            const int b = u.b, keys = u.keys, end = u.j1, y = u.kvh << plan.page_log2;
            last = u.flags & 1;
            // pages of key tile j that hold keys; this lane's page number, a tile ahead of its use
            const auto pages_in = [&](int j) { return max(0, min(ppt, (keys - j * 128 + page - 1) >> plan.page_log2)); };
            const int* row = plan.table + static_cast<long>(b) * plan.ld_table + my_page;
            const auto fetch = [&](int j) { return lane < boxes && my_page < pages_in(j) ? row[j * ppt] : 0; };
            int pg = fetch(u.j0);
            for (int j = u.j0; j < end; ++j, ++t) {
                const int n = pages_in(j) * S::HALVES;
                int cur = pg;
                if (j + 1 < end) pg = fetch(j + 1);
                bool w = true;
                if (lane == 0) {
                    w = mbar_wait(&empty[st], par, abort_flag, MICA_DEV_TIMEOUT_PRODUCER);
                    if (w) mbar_arrive_expect_tx(&full[st], n * box_bytes);
                }
                ok = __shfl_sync(0xffffffffu, w, 0);
                if (!ok) break;
                if (lane < n) {
                    // a page outside the pool is outside the map and reads as zeros
                    if (cur < 0 || cur >= plan.pages) { cur = plan.pages; record_bad_page(); }
                    tma_load_3d(ring + st * S::TILE + my_half * ATT_HALF_BYTES + my_page * box_bytes, map, &full[st], my_half * 64,
                                y, cur);
                }
                __syncwarp();
                if (++st == stages) { st = 0; par ^= 1u; }
            }
            if (!is_k && lane == 0) mbar_arrive(&unit_empty[slot]);
        }
        // the place of this CTA's last unit, for the join
        if (is_k && lane == 0) args.cuts[2 * cta + 1] = make_int4(unit > 1 ? 1 : 0, 0, 0, 0);
        // loads still in flight land before shared memory is released
        if (lane == 0) {
            if (is_k)
                for (int i = max(0, unit - S::QBUF); i < unit; ++i)
                    mbar_wait(&q_full[S::QBUF == 2 ? i & 1 : 0], i / S::QBUF & 1, abort_flag, MICA_DEV_TIMEOUT_DRAIN);
            for (int i = max(0, t - stages); i < t; ++i)
                mbar_wait(&full[i % stages], (i / stages) & 1, abort_flag, MICA_DEV_TIMEOUT_DRAIN);
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---------------------------------- MMA issuer --------------------------------
        // the whole warp, so that the operands' registers are uniform; one thread issues
        {
            const bool leader = elect_one();
            constexpr uint32_t idesc_qk = idesc_bf16(128, 128, false);
            constexpr uint32_t idesc_pv = idesc_bf16(128, D, true);
            const uint64_t q_desc0 = smem_desc_sw128(smem_u32(sq), 16, 1024);
            const uint64_t k_desc0 = smem_desc_sw128(smem_u32(sk), 16, 1024);
            const uint64_t v_desc0 = smem_desc_sw128(smem_u32(sv), ATT_HALF_BYTES, 1024);
            constexpr uint64_t kStep = S::TILE >> 4;
            bool ok = true, last = false;
            int t = 0, unit = 0;                  // tiles with scores issued, units
            int kst = 0, vst = 0, pv = 0;         // ring stages, tiles with P.V issued
            int fills = 0, pv1 = 0;               // NT 2: score tiles issued, P.V of row tile 1
            uint32_t kpar = 0u, vpar = 0u;
            const auto wait = [&](uint64_t* bar, uint32_t parity) {
                return __all_sync(0xffffffffu, mma_wait(bar, parity, abort_flag, MICA_DEV_TIMEOUT_MMA));
            };
            // scores of row tile x with the tile in kst, Q in buffer qb
            const auto scores = [&](int x, int qb) {
                const int i = NT == 1 ? (t & 1) : x;
                if (NT == 1) {
                    if (t >= 2 && !wait(&s_free[i], ((t >> 1) - 1) & 1)) return false;
                } else {
                    if (fills > 0 && !wait(&s_free[0], (fills - 1) & 1)) return false;
                    ++fills;
                }
                tc_fence_after();
                const uint64_t qd = q_desc0 + static_cast<uint64_t>(qb * NT + x) * kStep;
                const uint64_t kd = k_desc0 + static_cast<uint64_t>(kst) * kStep;
                if (leader) {
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint64_t off = static_cast<uint64_t>(((kk >> 2) * ATT_HALF_BYTES + (kk & 3) * 32) >> 4);
                        mma_bf16_ss(tmem + col_s(i), qd + off, kd + off, idesc_qk, kk > 0 ? 1u : 0u);
                    }
                    mma_commit(&s_full[i]);
                }
                return true;
            };
            int fixes = 0;                        // special tiles of the units before
            const auto values = [&](int x, bool fresh, bool special) {
                const int i = NT == 1 ? (pv & 1) : x;
                if (!wait(&p_full[i], (NT == 1 ? pv >> 1 : x ? pv1 : pv) & 1)) return false;
                if (NT == 2) pv1 += x;
                tc_fence_after();
                const uint64_t vd = v_desc0 + static_cast<uint64_t>(vst) * kStep;
                const uint32_t o = tmem + col_o(x), p = tmem + col_p(i);
                // the unit's first tile starts the accumulator, except where the softmax has put odd values there
                const bool start = fresh && !(special && cache_any_odd<NT>(odd_v, fixes));
                if (leader) {
                    mma_bf16_ts(o, p, vd, idesc_pv, start ? 0u : 1u);
#pragma unroll
                    for (int kk = 1; kk < 8; ++kk) mma_bf16_ts(o, p + kk * 8, vd + ((kk * 16 * 128) >> 4), idesc_pv, 1u);
                    mma_commit(&pv_done[i]);
                }
                return true;
            };
            const auto v_ready = [&]() { return wait(&v_full[vst], vpar); };
            const auto v_release = [&]() {
                if (leader) mma_commit(&v_empty[vst]);
                if (++vst == S::VST) { vst = 0; vpar ^= 1u; }
                ++pv;
            };
            // Inside a unit the scores of a tile are issued before the P.V of the tile before it. At its end the
            // rows are waited for, and the next unit's Q and K may be a while coming.
            for (; !last; ++unit) {
                const int qb = S::QBUF == 2 ? unit & 1 : 0;
                if (!wait(&unit_full[unit % CACHE_UNITS], unit / CACHE_UNITS & 1) ||
                    !wait(&q_full[qb], unit / S::QBUF & 1)) break;
                const volatile CacheUnit& u = units[unit % CACHE_UNITS];
                const int n = u.j1 - u.j0;
                bool fresh = true;
                const bool special = u.j0 >= u.special;                // its first tile is
                const int specials = max(0, u.j1 - max(u.j0, u.special));
                last = u.flags & 1;
                const auto tiles = [&](auto two) {
                    constexpr bool both = decltype(two)::value;
                    for (int j = 0; j < n; ++j, ++t) {
                        if (!wait(&k_full[kst], kpar) || !scores(0, qb)) return false;
                        if (!both && leader) mma_commit(&k_empty[kst]);
                        if (j > 0 && !(v_ready() && values(0, fresh, special))) return false;
                        if (both) {
                            if (!scores(1, qb)) return false;
                            if (leader) mma_commit(&k_empty[kst]);
                            if (j > 0 && !values(1, fresh, special)) return false;
                        }
                        if (++kst == S::KST) { kst = 0; kpar ^= 1u; }
                        if (j > 0) {
                            v_release();
                            fresh = false;
                        }
                    }
                    if (leader) mma_commit(&q_empty[qb]);
                    if (!v_ready() || !values(0, fresh, special) || (both && !values(1, fresh, special))) return false;
                    v_release();
                    return true;
                };
                if (NT == 2 && !(u.flags & 8)) ok = tiles(std::true_type());
                else ok = tiles(std::false_type());
                if (!ok) break;
                if (leader) mbar_arrive(&unit_empty[unit % CACHE_UNITS]);
                fixes += specials;
            }
            if (leader) mma_commit(drain);
            mbar_wait(drain, 0, abort_flag, MICA_DEV_TIMEOUT_DRAIN);
        }
        __syncwarp();
    } else if (warp == 3) {
        const bool ordered = cache_ordered(plan);
        if (lane == 0) {
            // the unit this CTA starts inside, for the join: its first row, node rows, K/V head, and the CTAs
            // that hold parts of it, the one before and `n` from this one on
            int4 cut = make_int4(0, 0, 0, ordered ? 0 : -1);
            if (ordered && wk.j0 > 0) {
                // places of the unit before each CTA's run: up to its first tile, up to its last
                const long first = static_cast<long>(Cost::UNIT) * wk.w, last = static_cast<long>(wk.nk - 1 + Cost::UNIT) * wk.w;
                const long unit0 = share.at(cta + 1) - wk.left;
                if (share.at(cta - 1) - unit0 <= first) {
                    int n = 1;
                    while (cta + n < share.used && share.at(cta + n) - unit0 <= last) ++n;
                    cut = make_int4(min(R, wk.s.T - wk.rb * R) * args.G, wk.s.row0 + wk.rb * R, wk.kvh, n);
                }
            }
            args.cuts[2 * cta] = cut;
        }
    } else {
        // ---------------------------------- softmax ----------------------------------
        const int x = (warp - 4) >> 2;                     // row tile of this warpgroup
        const int q4 = warp & 3;                           // tensor-memory lane quarter
        const uint32_t lane_off = static_cast<uint32_t>(q4 * 32) << 16;
        const float c = args.scale_log2;
        // in quarters each copy of the rows has 32 keys of a tile: this thread's row, its keys' first and number
        const int r = quarters ? lane : q4 * 32 + lane, key0 = quarters ? q4 * 32 : 0, keys_each = quarters ? 32 : 128;
        if (quarters) {                                    // the weights of the others' keys stay zero
            uint32_t zero[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) zero[i] = 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) tmem_st_32x32b_x32(tmem + col_p(0) + i * 32 + lane_off, zero);
            tmem_st_wait();
        }
        bool ok = true, last = false;
        int t = 0, unit = 0;                               // this row tile's key tiles so far, units
        int skipped = 0;                                   // and those of units it had no rows in
        int fixes = 0;                                     // special tiles so far
        for (; !last && ok; ++unit) {
            ok = __all_sync(0xffffffffu, mma_wait(&unit_full[unit % CACHE_UNITS], unit / CACHE_UNITS & 1, abort_flag,
                                                  MICA_DEV_TIMEOUT_EPILOGUE));
            if (!ok) break;
            const volatile CacheUnit& u = units[unit % CACHE_UNITS];
            last = u.flags & 1;
            const bool warp_live = r - lane < (u.nodes - x * args.npt) * args.G;   // some thread of the warp has a row
            const int t_first = t, t_end = t + u.j1 - u.j0, t_special = max(t, t + u.special - u.j0);
            if (NT == 2 && x == 1 && (u.flags & 8)) {                 // no rows: row tile 0 goes on alone
                skipped += t_end - t_first;
                fixes += max(0, t_end - t_special);
                __syncwarp();
                if (lane == 0) mbar_arrive(&unit_empty[unit % CACHE_UNITS]);
                continue;
            }
            const int node_r = r / args.G, head_r = r - node_r * args.G;
            const bool live = node_r < min(args.npt, u.nodes - x * args.npt);             // this thread has a row
            const uint32_t t_o = tmem + col_o(x) + lane_off;
            float m_use = CACHE_NOTHING, cr = c, l = 0.f;
            for (; t < t_end; ++t) {
                const int i2 = NT == 1 ? (t & 1) : x;
                const int n2 = NT == 1 ? t >> 1 : t;                   // uses of that buffer before
                const uint32_t t_s = tmem + col_s(i2) + lane_off, t_p = tmem + col_p(i2) + lane_off;
                const bool special = t >= t_special;
                ok = __all_sync(0xffffffffu, mma_wait(&s_full[i2], n2 & 1, abort_flag, MICA_DEV_TIMEOUT_EPILOGUE));
                if (!ok) break;
                tc_fence_after();
                // Only now, with the tile's scores: they were issued after the P.V of the tile two before, so V's
                // ring stage has had its last turn and its barrier's parity says whether this one's is over.
                if (special) {
                    const int vt = t + skipped;
                    ok = cache_safe_v<D, NT>(sv + vt % S::VST * S::TILE, &v_full[vt % S::VST], (vt / S::VST) & 1, v_fixed,
                                             odd_v + (fixes & 1) * NT * 4, u, (u.j0 + t - t_first) * 128, x, abort_flag);
                    if (!ok) break;
                }
                bool moved = false;                                  // the running maximum of a row
                float alpha = 1.f;
                uint32_t pk[64];
                // keys key0 .. of the tile, 32 W of them: weights into pk, row maximum and sum
                const auto weights = [&](auto part) {
                    constexpr int W = decltype(part)::value;
                    uint32_t sr[32 * W];
#pragma unroll
                    for (int cc = 0; cc < W; ++cc)
                        tmem_ld_32x32b_x32(t_s + key0 + cc * 32, *reinterpret_cast<uint32_t (*)[32]>(&sr[cc * 32]));
                    tmem_ld_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_free[NT == 1 ? i2 : 0]);
                    if (special) {
                        uint32_t vis[4];
                        cache_visible(args, u, x, node_r, (u.j0 + t - t_first) * 128 + key0, vis);
#pragma unroll
                        for (int i = 0; i < 32 * W; ++i)
                            if (!(vis[i >> 5] >> (i & 31) & 1u)) sr[i] = 0xff800000u;
                    }
                    float mp[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        mp[e] = fmax3(__uint_as_float(sr[e]), __uint_as_float(sr[8 + e]), __uint_as_float(sr[16 + e]));
#pragma unroll
                    for (int i = 24; i < 32 * W; i += 16)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            mp[e] = i + 8 + e < 32 * W ? fmax3(mp[e], __uint_as_float(sr[i + e]), __uint_as_float(sr[i + 8 + e]))
                                                       : fmaxf(mp[e], __uint_as_float(sr[i + e]));
                    const float mx = fmax3(fmax3(mp[0], mp[1], mp[2]), fmax3(mp[3], mp[4], mp[5]), fmaxf(mp[6], mp[7]));
                    if (fmaf(mx, cr, -m_use) > ATT_RESCALE_LOG2) {
                        float m_new = mx * c;
                        cr = c;
                        if (fabsf(m_new) > CACHE_FAR) {
                            cr = __uint_as_float((__float_as_uint(c) + 0x007fffffu) & 0x7f800000u);
                            m_new = mx * cr;
                        }
                        alpha = fast_exp2(m_use - m_new);
                        m_use = m_new;
                        moved = live;                // what a thread without a row reads and adds up is nobody's
                    }
                    const unsigned long long c2 = f2_pack(cr, cr), nm2 = f2_pack(-m_use, -m_use);
                    unsigned long long sp[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
                    for (int i = 0; i < 16 * W; ++i) {
                        const unsigned long long x2 =
                            f2_fma(f2_pack(__uint_as_float(sr[2 * i]), __uint_as_float(sr[2 * i + 1])), c2, nm2);
                        float x0, x1;
                        f2_unpack(x2, x0, x1);
                        const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
                        sp[i & 3] = f2_add(sp[i & 3], f2_pack(p0, p1));
                        pk[i] = pack_bf16(p0, p1);
                    }
                    float a0, a1, b0, b1, d0, d1, e0, e1;
                    f2_unpack(sp[0], a0, a1);
                    f2_unpack(sp[1], b0, b1);
                    f2_unpack(sp[2], d0, d1);
                    f2_unpack(sp[3], e0, e1);
                    l = l * alpha + (((a0 + a1) + (b0 + b1)) + ((d0 + d1) + (e0 + e1)));
                };
                if (warp_live) {
                    if (!quarters) weights(std::integral_constant<int, 4>());
                    else weights(std::integral_constant<int, 1>());
                } else {
                    if (lane == 0) mbar_arrive(&s_free[NT == 1 ? i2 : 0]);
                }
                // this P buffer is free once its last P.V is done; the accumulator once the tile before's is
                bool any_odd = false;
                if (special) {
                    ok = __all_sync(0xffffffffu, mbar_wait(v_fixed, fixes & 1, abort_flag, MICA_DEV_TIMEOUT_EPILOGUE));
                    if (!ok) break;
                    any_odd = cache_any_odd<NT>(odd_v, fixes++);
                }
                const bool fresh = t == t_first;
                const bool touch = warp_live && (any_odd || (!fresh && __any_sync(0xffffffffu, moved)));
                // NT 1: the scores were issued after the P.V of the tile two before, and are there
                if (NT == 2 && n2 > 0)
                    ok = __all_sync(0xffffffffu, mma_wait(&pv_done[i2], (n2 - 1) & 1, abort_flag, MICA_DEV_TIMEOUT_EPILOGUE));
                if (NT == 1 && touch && t >= 1)
                    ok = __all_sync(0xffffffffu, mma_wait(&pv_done[i2 ^ 1], ((t - 1) >> 1) & 1, abort_flag, MICA_DEV_TIMEOUT_EPILOGUE));
                if (!ok) break;
                if (NT == 2 || touch) tc_fence_after();
                if (touch) {
#pragma unroll 1
                    for (int cc = 0; cc < D / 32; ++cc) {
                        uint32_t o[32];
                        if (fresh) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = 0u;
                        } else {
                            tmem_ld_32x32b_x32(t_o + cc * 32, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        }
                        if (any_odd) {
                            const volatile uint32_t* odd4 = odd_v + (~fixes & 1) * 4 * NT;      // counted already
                            const int k0 = (u.j0 + t - t_first) * 128;
                            uint32_t vis[4];
                            cache_visible(args, u, x, node_r, k0, vis);
#pragma unroll 1
                            for (int i = key0; i < key0 + keys_each; ++i) {
                                const uint32_t bit = 1u << (i & 31);
                                const uint32_t seen = i < 64 ? (i < 32 ? vis[0] : vis[1]) : (i < 96 ? vis[2] : vis[3]);
                                int pgn = 0, slot = 0;
                                if (!((odd4[i >> 5] | odd4[(NT - 1) * 4 + (i >> 5)]) & bit) || !(seen & bit) ||
                                    !cache_slot(plan, u.b, k0 + i, &pgn, &slot)) continue;
                                const uint16_t* v = reinterpret_cast<const uint16_t*>(args.v_pages) + pgn * args.page_stride +
                                                    ((static_cast<long>(u.kvh) << plan.page_log2) + slot) * D + cc * 32;
#pragma unroll
                                for (int e = 0; e < 32; ++e) {
                                    const uint32_t bits = v[e];
                                    if ((bits & 0x7f80u) == 0x7f80u)
                                        o[e] = __float_as_uint(__uint_as_float(o[e]) + __uint_as_float(bits << 16));
                                }
                            }
                        }
                        __syncwarp();
                        tmem_st_32x32b_x32(t_o + cc * 32, o);
                    }
                }
                if (warp_live) {
                    if (quarters) {
                        tmem_st_32x32b_x16(t_p + key0 / 2, *reinterpret_cast<uint32_t (*)[16]>(&pk[0]));
                    } else {
                        tmem_st_32x32b_x32(t_p, *reinterpret_cast<uint32_t (*)[32]>(&pk[0]));
                        tmem_st_32x32b_x32(t_p + 32, *reinterpret_cast<uint32_t (*)[32]>(&pk[32]));
                    }
                    tmem_st_wait();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[i2]);
            }
            if (!ok) break;
            // the unit's rows: out, or this CTA's place in the workspace
            {
                const int tl = t - 1;
                const int i2 = NT == 1 ? (tl & 1) : x;
                const int n2 = NT == 1 ? tl >> 1 : tl;
                ok = __all_sync(0xffffffffu, mma_wait(&pv_done[i2], n2 & 1, abort_flag, MICA_DEV_TIMEOUT_EPILOGUE));
                if (!ok) break;
                tc_fence_after();
                const bool whole = u.flags & 2;
                const long row = static_cast<long>(u.row0) + x * args.npt + node_r;
                float* place = args.ws + (cta * 2l + (u.flags & 4 ? 0 : 1)) * cache_attn_place_floats<D, NT>();
                float4* part = reinterpret_cast<float4*>(place) + x * (D / 4) * 128 + r;
                float2* part_ml = reinterpret_cast<float2*>(place + NT * 128l * D) + x * 128 + r;
                __nv_bfloat16* orow = args.out + row * args.ldo + (u.kvh * args.G + head_r) * D;
                if (quarters) {
                    // The copies, brought to one maximum and added up through the unit's Q buffer (their 4 * 16
                    // rows at most fill it): the four warps share the (row, 4 columns).
                    const int rows = args.npt * args.G, have = min(args.npt, u.nodes) * args.G;   // of a copy; of the unit
                    float4* xo = reinterpret_cast<float4*>(sq + (unit & 1) * S::TILE);            // [copy][D / 4][rows]
                    if (live) stats[q4 * 32 + r] = make_float2(m_use, l);
#pragma unroll
                    for (int cc = 0; cc < D / 32; ++cc) {
                        uint32_t o[32];
                        tmem_ld_32x32b_x32(t_o + cc * 32, o);
                        tmem_ld_wait();
                        if (live) {
#pragma unroll
                            for (int v = 0; v < 8; ++v)
                                xo[(q4 * (D / 4) + cc * 8 + v) * rows + r] =
                                    make_float4(__uint_as_float(o[4 * v]), __uint_as_float(o[4 * v + 1]),
                                                __uint_as_float(o[4 * v + 2]), __uint_as_float(o[4 * v + 3]));
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(exchange);
                    ok = __all_sync(0xffffffffu, mma_wait(exchange, unit & 1, abort_flag, MICA_DEV_TIMEOUT_EPILOGUE));
                    if (!ok) break;
                    for (int i0 = q4 * 32; i0 < D / 4 * rows; i0 += 128) {
                        const int item = i0 + lane, v = min(item / rows, D / 4 - 1), rr = item - v * rows;
                        const bool mine = rr < have;
                        float m_all = CACHE_NOTHING, l_all = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
                        if (mine) {
                            float2 ml[4];
                            float4 a[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                ml[k] = stats[k * 32 + rr];
                                a[k] = xo[(k * (D / 4) + v) * rows + rr];
                            }
#pragma unroll
                            for (int k = 0; k < 4; ++k) m_all = fmaxf(m_all, ml[k].x);
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const float w = fast_exp2(ml[k].x - m_all);
                                l_all = fmaf(ml[k].y, w, l_all);
                                o[0] = fmaf(a[k].x, w, o[0]);
                                o[1] = fmaf(a[k].y, w, o[1]);
                                o[2] = fmaf(a[k].z, w, o[2]);
                                o[3] = fmaf(a[k].w, w, o[3]);
                            }
                        }
                        const int node = rr / args.G;
                        float zero = 0.f;
#pragma unroll
                        for (int e = 0; e < 4; ++e) zero = fmaf(o[e], 0.f, zero);
                        const bool odd = zero != 0.f && l_all * 0.f == 0.f;           // infinite or NaN scores stay
                        if (__any_sync(0xffffffffu, odd)) {
                            const uint32_t kinds = cache_odd_kinds<D>(args, u, node, v * 4, odd);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const uint32_t n = kinds >> (3 * e) & 7u;
                                if (n) o[e] = __uint_as_float(n & 1u || n == 6u ? 0x7fffffffu : n == 2u ? 0x7f800000u : 0xff800000u);
                            }
                        }
                        if (mine && whole) {
                            const float inv = l_all == 0.f ? 0.f : 1.f / l_all;
                            *reinterpret_cast<uint2*>(args.out + (static_cast<long>(u.row0) + node) * args.ldo +
                                                      (u.kvh * args.G + rr - node * args.G) * D + v * 4) =
                                make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
                        } else if (mine) {
                            reinterpret_cast<float4*>(place)[v * 128 + rr] = make_float4(o[0], o[1], o[2], o[3]);
                            if (v == 0) reinterpret_cast<float2*>(place + 128l * D)[rr] = make_float2(m_all, l_all);
                        }
                    }
                    fence_proxy_async_smem();                        // Q of the next unit but one comes here
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&q_empty[unit & 1]);
                } else if (warp_live) {
                    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
                    for (int cc = 0; cc < D / 32; ++cc) {
                        uint32_t o[32];
                        tmem_ld_32x32b_x32(t_o + cc * 32, o);
                        tmem_ld_wait();
                        if (live && whole) {
#pragma unroll
                            for (int v = 0; v < 4; ++v) {
                                uint4 pkt;
                                pkt.x = pack_bf16(__uint_as_float(o[8 * v + 0]) * inv, __uint_as_float(o[8 * v + 1]) * inv);
                                pkt.y = pack_bf16(__uint_as_float(o[8 * v + 2]) * inv, __uint_as_float(o[8 * v + 3]) * inv);
                                pkt.z = pack_bf16(__uint_as_float(o[8 * v + 4]) * inv, __uint_as_float(o[8 * v + 5]) * inv);
                                pkt.w = pack_bf16(__uint_as_float(o[8 * v + 6]) * inv, __uint_as_float(o[8 * v + 7]) * inv);
                                *reinterpret_cast<uint4*>(orow + cc * 32 + v * 8) = pkt;
                            }
                        } else if (live) {
#pragma unroll
                            for (int v = 0; v < 8; ++v)
                                part[(cc * 8 + v) * 128] = make_float4(__uint_as_float(o[4 * v]), __uint_as_float(o[4 * v + 1]),
                                                                       __uint_as_float(o[4 * v + 2]), __uint_as_float(o[4 * v + 3]));
                        }
                    }
                    if (live && !whole) *part_ml = make_float2(m_use, l);
                    tc_fence_before();
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&unit_empty[unit % CACHE_UNITS]);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_free(tmem, 512);
    }
    cache_zero_padding(args, D, threadIdx.x, blockDim.x);
}

// Adds up the parts of each divided unit, always in the same order. Blocks (c, y): the unit that CTA c + 1 is
// the first to start inside, if it is. A thread takes 16 columns of a row, three parts in flight; where a
// long sequence's unit is in many parts, `lanes` neighbouring threads take every lanes-th part each and add
// theirs up (one sequence of 100000 keys and one K/V head is in 148: 35 us one part after the other).
// Where the row offsets were out of order it makes all rows zero.
__host__ __device__ inline int cache_join_lanes(int parts) { return parts < 6 ? 1 : parts < 24 ? 4 : 16; }
template <int D, int NT>
__global__ void __launch_bounds__(128) cache_attention_join(const CacheAttnArgs args) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int AHEAD = 3;
    const int c = blockIdx.x + 1;
    const int4 cut = args.cuts[2 * c];
    const int rows = cut.x, n = cut.w, items = rows * (D / 16);
    if (items == 0) {
        if (n < 0)
            cache_zero_rows(args, D, 0, 0, static_cast<long>(blockIdx.y) * gridDim.x + blockIdx.x,
                            static_cast<long>(gridDim.x) * gridDim.y, threadIdx.x, blockDim.x);
        return;
    }
    const int lanes = cache_join_lanes(n);
    const int first_place = args.cuts[2 * (c - 1) + 1].x;            // of the part that the CTA before left last
    const long pf = cache_attn_place_floats<D, NT>();
    const float* part0 = args.ws + ((c - 1) * 2l + first_place) * pf;
    const float* parts = args.ws + c * 2l * pf;
    const int mine = threadIdx.x % lanes, groups = gridDim.y * blockDim.x / lanes;
    // whole warps go round together: an item behind the last is the last once more, not written
    for (int i0 = (blockIdx.y * blockDim.x + (threadIdx.x & ~31)) / lanes; i0 < items; i0 += groups) {
        const int item = i0 + (threadIdx.x & 31) / lanes, idx = min(item, items - 1);
        const int rr = idx % rows, d16 = idx / rows;
        const int node = rr / args.G, g = rr - node * args.G;
        const int x = NT == 1 ? 0 : node / args.npt, r = (node - x * args.npt) * args.G + g;
        float m = -INFINITY, l = 0.f;
        float4 o[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) o[v] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int p0 = mine; p0 <= n; p0 += AHEAD * lanes) {
            float2 ml[AHEAD];
            float4 p[AHEAD][4];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int i = p0 + u * lanes;
                if (i > n) continue;
                const float* a = i == 0 ? part0 : parts + (i - 1) * 2l * pf;
                ml[u] = __ldcg(reinterpret_cast<const float2*>(a + NT * 128l * D) + x * 128 + r);
#pragma unroll
                for (int v = 0; v < 4; ++v) p[u][v] = __ldcg(reinterpret_cast<const float4*>(a) + (x * (D / 4) + d16 * 4 + v) * 128 + r);
            }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                if (p0 + u * lanes > n) continue;
                const float mn = fmaxf(m, ml[u].x), wo = fast_exp2(m - mn), w = fast_exp2(ml[u].x - mn);
                m = mn;
                l = fmaf(ml[u].y, w, l * wo);
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    o[v].x = fmaf(p[u][v].x, w, o[v].x * wo);
                    o[v].y = fmaf(p[u][v].y, w, o[v].y * wo);
                    o[v].z = fmaf(p[u][v].z, w, o[v].z * wo);
                    o[v].w = fmaf(p[u][v].w, w, o[v].w * wo);
                }
            }
        }
        for (int s = 1; s < lanes; s <<= 1) {
            const float mo = __shfl_xor_sync(0xffffffffu, m, s), mn = fmaxf(m, mo);
            const float w = m == -INFINITY ? 0.f : fast_exp2(m - mn);                  // -inf: no part
            const auto add = [&](float f) {
                f = m == -INFINITY ? 0.f : f * w;
                return f + __shfl_xor_sync(0xffffffffu, f, s);
            };
            l = add(l);
#pragma unroll
            for (int v = 0; v < 4; ++v) o[v] = make_float4(add(o[v].x), add(o[v].y), add(o[v].z), add(o[v].w));
            m = mn;
        }
        if (mine || item >= items) continue;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const long row = static_cast<long>(cut.y) + node;
        uint4* to = reinterpret_cast<uint4*>(args.out + row * args.ldo + (cut.z * args.G + g) * D + d16 * 16);
#pragma unroll
        for (int v = 0; v < 4; v += 2)
            to[v / 2] = make_uint4(pack_bf16(o[v].x * inv, o[v].y * inv), pack_bf16(o[v].z * inv, o[v].w * inv),
                                   pack_bf16(o[v + 1].x * inv, o[v + 1].y * inv), pack_bf16(o[v + 1].z * inv, o[v + 1].w * inv));
    }
}

}  // namespace mica
