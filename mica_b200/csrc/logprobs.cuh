// logprobs.cuh -- log probabilities of given tokens, entropy and top alternatives of logits rows.
//
//   m = max_v z_v,  S = sum_v e^(z_v - m),  lse = m + log S
//   logprob[r, j] = z[r, ids[r, j]] - lse        (a negative id is padding: 0; one past the end: NaN)
//   entropy[r]    = log S + sum_v (m - z_v) e^(z_v - m) / S          (a sum of terms >= 0)
//   top[r, j]     = the j-th largest z - lse and its id, ties to the lowest id, NaN before all
// A row whose logits are all -inf allows nothing: log probabilities -inf, entropy 0. A NaN or +inf
// logit makes the row NaN.
//
// Bound by the logits' bytes, which are read once: the maximum, S and the entropy's sum run along in
// one pass (rescaled when the maximum grows), in base 2 and fp32. A row is one cluster of CTAs, each
// with a run of it; the parts meet through distributed shared memory, so there is one launch and
// no workspace.
//
// Alternatives without a list in the inner loop: a thread keeps only the largest logit it has seen.
// The CTA's 32 half-warps give 32 maxima of disjoint elements, so the top-th largest of those is a
// lower bound of the run's top-th largest logit; only threads whose maximum reaches it can hold an
// alternative, about one in sixteen, and their elements are read again (from L2) and kept when they
// reach the bound: about 30 candidates for 20 alternatives of random logits. They are ranked by
// counting, in each CTA and then over the cluster.
#pragma once

#include "quant.cuh"

namespace mica {

struct LogprobArgs {
    const void* z;              // [N, ld]
    long ld;
    int N, V;
    const long* ids;            // [N, ld_ids]
    long ld_ids;
    int M, top;
    float* logprob;             // [N, M]
    float* entropy;             // [N]
    float* top_lp;              // [N, top]
    long* top_id;               // [N, top]
};

constexpr int LP_THREADS = 512;
constexpr int LP_WARPS = LP_THREADS / 32;
constexpr int LP_UNROLL = 4;             // 16-byte vectors a thread has in flight
constexpr int LP_CAND = 1024;            // candidates a CTA can rank
constexpr int LP_TOP = 32;
constexpr int LP_CLUSTER = 16;
static_assert(2 * LP_WARPS == LP_TOP, "one group maximum for each alternative");
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Logits are held above this in the sums, so that a weight of zero meets no infinity; a row whose
// maximum is not well above it (or is beyond its negative) is computed again without the limit.
constexpr float LP_FLOOR = -1e38f;

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
    if constexpr (std::is_same<T, float>::value) return v;
    else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
    else return __bfloat162float(v);
}
__device__ __forceinline__ float nan_f32() { return __uint_as_float(0x7fc00000u); }

// Orders logits for the alternatives: larger value first, NaN above +inf, -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float z) {
    if (z != z) return 0xffffffffu;
    const uint32_t u = __float_as_uint(z + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t k) {
    if (k == 0xffffffffu) return nan_f32();
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ unsigned long long rank_key(float z, int id) {
    return static_cast<unsigned long long>(order_key(z)) << 32 | ~static_cast<uint32_t>(id);
}

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Sums of a set of logits in base 2: mc = log2(e) * (its maximum), s = sum 2^(z log2e - mc),
// w = sum (z log2e - mc) 2^(z log2e - mc). z log2e - mc is one fma with the same mc everywhere, so
// the rounding of mc cancels between the sums and z - lse.
struct LpSums {
    float mc, s, w;
};
__device__ __forceinline__ LpSums lp_join(const LpSums& a, const LpSums& b) {
    const float mc = max_nan(a.mc, b.mc);
    const float da = fmaxf(a.mc - mc, -1000.f), db = fmaxf(b.mc - mc, -1000.f);    // 2^-1000 is 0, its product too
    const float fa = exp2f(da), fb = exp2f(db);
    return LpSums{mc, a.s * fa + b.s * fb, fa * fmaf(da, a.s, a.w) + fb * fmaf(db, b.s, b.w)};
}

// The 16-byte vector's values.
template <typename T>
struct LpVec {
    static constexpr int N = 16 / sizeof(T);
    __device__ __forceinline__ static void values(const uint4& q, float (&f)[N]) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                f[i] = __uint_as_float(w[i]);
            } else if constexpr (std::is_same<T, __half>::value) {
                const __half2 h = *reinterpret_cast<const __half2*>(&w[i]);
                f[2 * i] = __low2float(h);
                f[2 * i + 1] = __high2float(h);
            } else {
                f[2 * i] = __uint_as_float(w[i] << 16);
                f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
};

// One thread's step: its sums and largest logit take in LP_UNROLL vectors.
template <typename T>
__device__ __forceinline__ void lp_step(const uint4 (&q)[LP_UNROLL], LpSums& a, float& top) {
    constexpr int N = LpVec<T>::N;
    float cm;
    uint4 c[LP_UNROLL];
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {       // maxima of pairs
        __nv_bfloat162 m2 = *reinterpret_cast<const __nv_bfloat162*>(&q[0].x);
        const __nv_bfloat162 lo2 = __float2bfloat162_rn(LP_FLOOR);
#pragma unroll
        for (int u = 0; u < LP_UNROLL; ++u) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(&q[u]);
            uint32_t* o = reinterpret_cast<uint32_t*>(&c[u]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&w[i]);
                m2 = __hmax2_nan(m2, v);
                const __nv_bfloat162 l = __hmax2_nan(v, lo2);
                o[i] = *reinterpret_cast<const uint32_t*>(&l);
            }
        }
        cm = max_nan(__low2float(m2), __high2float(m2));
    } else {
        float f[N];
        cm = -INFINITY;
#pragma unroll
        for (int u = 0; u < LP_UNROLL; ++u) {
            LpVec<T>::values(q[u], f);
#pragma unroll
            for (int i = 0; i < N; ++i) cm = max_nan(cm, f[i]);
            c[u] = q[u];
        }
    }
    top = max_nan(top, cm);
    const float cmc = max_nan(cm, LP_FLOOR) * kLog2e;
    if (!(cmc <= a.mc)) {
        const float d = fmaxf(a.mc - cmc, -1000.f), f = exp2f(d);
        a.w = f * fmaf(d, a.s, a.w);
        a.s *= f;
        a.mc = cmc;
    }
    const unsigned long long c2 = f2_pack(kLog2e, kLog2e), n2 = f2_pack(-a.mc, -a.mc);
    unsigned long long s2 = 0ull, w2 = 0ull;
#pragma unroll
    for (int u = 0; u < LP_UNROLL; ++u) {
        float f[N];
        LpVec<T>::values(c[u], f);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            if constexpr (!std::is_same<T, __nv_bfloat16>::value) {
                f[i] = max_nan(f[i], LP_FLOOR);
                f[i + 1] = max_nan(f[i + 1], LP_FLOOR);
            }
            const unsigned long long d2 = f2_fma(f2_pack(f[i], f[i + 1]), c2, n2);
            float d0, d1;
            f2_unpack(d2, d0, d1);
            const unsigned long long e2 = f2_pack(fast_exp2(d0), fast_exp2(d1));
            s2 = f2_add(s2, e2);
            w2 = f2_fma(d2, e2, w2);
        }
    }
    float x, y;
    f2_unpack(s2, x, y);
    a.s += x + y;
    f2_unpack(w2, x, y);
    a.w += x + y;
}

struct LpPart {                 // what a CTA tells its cluster
    LpSums sums;
    int count;                  // entries of list
    unsigned long long list[LP_TOP];
};

// The whole row by one CTA, in passes, for rows beyond the sums' range (infinities, NaN, maxima
// near the type's ends) : the definition literally.
template <typename T>
__device__ void lp_row_plain(const LogprobArgs& a, const T* z, float* red, float& m, float& logs, float& ent) {
    m = -INFINITY;
    bool odd = false;
    for (int i = threadIdx.x; i < a.V; i += LP_THREADS) {
        const float v = to_f32(z[i]);
        odd |= v != v || v == INFINITY;
        m = fmaxf(m, v);
    }
    odd = __syncthreads_or(odd);
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int i = 0; i < LP_WARPS; ++i) m = fmaxf(m, red[i]);
    __syncthreads();
    float s = 0.f, w = 0.f;
    for (int i = threadIdx.x; i < a.V; i += LP_THREADS) {
        const float d = to_f32(z[i]) - m, e = m == -INFINITY ? 0.f : expf(d);
        s += e;
        if (e > 0.f) w -= d * e;
    }
    s = block_reduce<false>(s, red);
    w = block_reduce<false>(w, red);
    logs = m == -INFINITY ? 0.f : logf(s);
    ent = m == -INFINITY ? 0.f : logs + w / s;
    if (odd) logs = ent = nan_f32();
}

// Elements [i0, i1) of the row, each alternative by one pass: for runs with more ties than a list holds.
template <typename T>
__device__ void lp_select_plain(const T* z, int i0, int i1, int top, unsigned long long* list, unsigned long long* best) {
    unsigned long long last = ~0ull;
    for (int j = 0; j < top; ++j) {
        unsigned long long b = 0ull;
        for (int i = i0 + threadIdx.x; i < i1; i += LP_THREADS) {
            const unsigned long long c = rank_key(to_f32(z[i]), i);
            if (c < last && c > b) b = c;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long c = __shfl_xor_sync(0xffffffffu, b, o);
            b = c > b ? c : b;
        }
        __syncthreads();
        if ((threadIdx.x & 31) == 0) best[threadIdx.x >> 5] = b;
        __syncthreads();
        for (int i = 0; i < LP_WARPS; ++i) b = best[i] > b ? best[i] : b;
        last = b;
        if (threadIdx.x == 0) list[j] = b;
    }
    __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS, 2) token_logprobs_kernel(const LogprobArgs a, const int parts) {
    constexpr int N = LpVec<T>::N;
    __shared__ float red[32];
    __shared__ unsigned long long cand[LP_CAND];
    __shared__ LpPart part;
    __shared__ float s_group[LP_TOP], s_bound;
    __shared__ int s_count;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = parts > 1 ? static_cast<int>(cluster_ctarank()) : 0;
    const int row = blockIdx.x / parts;
    const T* z = static_cast<const T*>(a.z) + static_cast<long>(row) * a.ld;
    // [0, head) single elements up to the first 16-byte boundary, nvec vectors, single elements to V
    const int head = min(a.V, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / static_cast<int>(sizeof(T)));
    const int nvec = (a.V - head) / N;
    const uint4* zv = reinterpret_cast<const uint4*>(z + head);
    const int v0 = static_cast<int>(static_cast<long>(nvec) * rank / parts);
    const int v1 = static_cast<int>(static_cast<long>(nvec) * (rank + 1) / parts);
    // the single elements, fewer than N at either end, are the first and the last CTA's, one a thread
    const int tail = head + nvec * N, tid = threadIdx.x;
    const int my_loose = rank == 0 && tid < head                                       ? tid
                         : rank == parts - 1 && tid >= 16 && tail + (tid - 16) < a.V ? tail + (tid - 16) : -1;

    // ---- the pass ----
    constexpr uint32_t kNone = std::is_same<T, float>::value ? 0xff800000u
                               : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;    // -inf
    LpSums sums{LP_FLOOR * kLog2e, 0.f, 0.f};
    float top = -INFINITY;
    int v = v0 + threadIdx.x;
    for (; v + (LP_UNROLL - 1) * LP_THREADS < v1; v += LP_UNROLL * LP_THREADS) {
        uint4 q[LP_UNROLL];
#pragma unroll
        for (int u = 0; u < LP_UNROLL; ++u) q[u] = __ldg(zv + v + u * LP_THREADS);
        lp_step<T>(q, sums, top);
    }
    if (v < v1 || my_loose >= 0) {
        uint4 q[LP_UNROLL];
#pragma unroll
        for (int u = 0; u < LP_UNROLL; ++u)
            q[u] = v + u * LP_THREADS < v1 ? __ldg(zv + v + u * LP_THREADS) : make_uint4(kNone, kNone, kNone, kNone);
        lp_step<T>(q, sums, top);
        if (my_loose >= 0) {
            const float f = to_f32(z[my_loose]);
            top = max_nan(top, f);
            sums = lp_join(sums, LpSums{max_nan(f, LP_FLOOR) * kLog2e, 1.f, 0.f});
        }
    }

    // ---- alternatives of the run ----
    if (threadIdx.x == 0) s_count = 0;
    if (a.top > 0) {
        float g = top;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) g = max_nan(g, __shfl_xor_sync(0xffffffffu, g, o));
        if ((lane & 15) == 0) s_group[threadIdx.x >> 4] = g;
        __syncthreads();
        if (warp == 0) {
            // the top-th largest of the 32 maxima
            const uint32_t mine = order_key(s_group[lane]);
            int above = 0;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const uint32_t o = __shfl_sync(0xffffffffu, mine, i);
                above += o > mine || (o == mine && i < lane);
            }
            if (above == a.top - 1) s_bound = order_value(mine);
        }
        __syncthreads();
        const float bound = s_bound;
        const uint32_t bkey = order_key(bound);
        const int n_mine = v1 - v0;
        // elements that reach the bound (strict: that are above it)
        const auto gather = [&](bool strict) {
            const auto keep = [&](float f, int id) {
                const uint32_t k = order_key(f);
                if (strict ? k > bkey : k >= bkey) {
                    const int at = atomicAdd(&s_count, 1);
                    if (at < LP_CAND) cand[at] = rank_key(f, id);
                }
            };
            uint32_t who = __ballot_sync(0xffffffffu, order_key(top) >= bkey);
            for (; who; who &= who - 1) {
                // the warp reads that thread's vectors, one a lane
                const int t = warp * 32 + __ffs(who) - 1;
                for (int i = t + lane * LP_THREADS; i < n_mine; i += 32 * LP_THREADS) {
                    float f[N];
                    LpVec<T>::values(__ldg(zv + v0 + i), f);
#pragma unroll
                    for (int e = 0; e < N; ++e) keep(f[e], head + (v0 + i) * N + e);
                }
            }
            if (my_loose >= 0) keep(to_f32(z[my_loose]), my_loose);
        };
        gather(false);
        __syncthreads();
        int n = s_count;
        const int lo = rank == 0 ? 0 : head + v0 * N, hi = rank == parts - 1 ? a.V : head + v1 * N;   // the run's elements
        bool plain = false;
        if (n > LP_CAND) {
            // more ties at the bound than places (a row that allows few tokens, or equal logits): those above
            // it, then the first ones at it in order of their ids
            __syncthreads();
            if (threadIdx.x == 0) s_count = 0;
            __syncthreads();
            gather(true);
            __syncthreads();
            n = s_count;
            plain = n > LP_CAND - LP_TOP;
            const int want = plain ? 0 : n + a.top;              // enough of them
            for (int i0 = lo; i0 < hi && n < want; i0 += LP_THREADS) {
                const int i = i0 + threadIdx.x;
                const bool hit = i < hi && order_key(to_f32(z[i])) == bkey;
                const uint32_t bits = __ballot_sync(0xffffffffu, hit);
                __syncthreads();
                if (lane == 0) red[warp] = __uint_as_float(__popc(bits));
                __syncthreads();
                int at = n;
                for (int w = 0; w < LP_WARPS; ++w) {
                    const int k = __float_as_uint(red[w]);
                    if (w < warp) at += k;
                    n += k;
                }
                at += __popc(bits & ((1u << lane) - 1u));
                if (hit && at < want) cand[at] = rank_key(order_value(bkey), i);
                n = min(n, want);
            }
            __syncthreads();
        }
        if (plain) {
            lp_select_plain(z, lo, hi, a.top, part.list, cand);
            if (threadIdx.x == 0) part.count = min(a.top, hi - lo);
        } else {
            for (int i = threadIdx.x; i < n; i += LP_THREADS) {
                const unsigned long long k = cand[i];
                int above = 0;
                for (int j = 0; j < n; ++j) above += cand[j] > k;
                if (above < a.top) part.list[above] = k;
            }
            if (threadIdx.x == 0) part.count = min(n, a.top);
        }
    }

    // ---- sums of the run ----
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const LpSums b{__shfl_xor_sync(0xffffffffu, sums.mc, o), __shfl_xor_sync(0xffffffffu, sums.s, o),
                       __shfl_xor_sync(0xffffffffu, sums.w, o)};
        // the same order on both sides, so both get the same bits
        sums = lane & o ? lp_join(b, sums) : lp_join(sums, b);
    }
    __shared__ LpSums s_sums[LP_WARPS];
    if (lane == 0) s_sums[warp] = sums;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < LP_WARPS; ++i) sums = lp_join(sums, s_sums[i]);
        part.sums = sums;
    }

    // ---- the cluster's parts ----
    if (parts > 1) cluster_sync(); else __syncthreads();
    if (rank == 0) {
        const auto remote = [&](int r, const void* p) {
            return map_to_rank(smem_u32(p), r);
        };
        sums = part.sums;
        for (int r = 1; r < parts; ++r) {
            LpSums b;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b.mc) : "r"(remote(r, &part.sums.mc)) : "memory");
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b.s) : "r"(remote(r, &part.sums.s)) : "memory");
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b.w) : "r"(remote(r, &part.sums.w)) : "memory");
            sums = lp_join(sums, b);
        }
        int n = 0;
        if (a.top > 0) {
            // at most 16 x 32 candidates: one a thread
            const int r = threadIdx.x >> 5;
            unsigned long long k = 0ull;
            if (r < parts) {
                int count;
                asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(count) : "r"(remote(r, &part.count)) : "memory");
                if (lane < count)
                    asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(k) : "r"(remote(r, &part.list[lane])) : "memory");
            }
            cand[threadIdx.x] = k;
            n = parts * LP_TOP;
            __syncthreads();
        }
        const float log2s = log2f(sums.s);
        float m = 0.f, logs = 0.f, ent = kLn2 * (log2s - sums.w / sums.s);
        // beyond the range of the sums, or NaN
        const bool odd = !(sums.mc > 0.1f * LP_FLOOR && sums.mc < -LP_FLOOR && sums.s < INFINITY);
        if (odd) lp_row_plain(a, z, red, m, logs, ent);
        const auto lp = [&](float f) {
            if (odd) return m == -INFINITY && logs == 0.f ? -INFINITY : (f - m) - logs;
            return (fmaf(f, kLog2e, -sums.mc) - log2s) * kLn2;
        };
        if (threadIdx.x == 0) a.entropy[row] = ent;
        for (int j = threadIdx.x; j < a.M; j += LP_THREADS) {
            const long id = a.ids[static_cast<long>(row) * a.ld_ids + j];
            a.logprob[static_cast<long>(row) * a.M + j] = id < 0 ? 0.f : id >= a.V ? nan_f32() : lp(to_f32(z[id]));
        }
        if (static_cast<int>(threadIdx.x) < n && cand[threadIdx.x]) {
            const unsigned long long k = cand[threadIdx.x];
            int above = 0;
            for (int j = 0; j < n; ++j) above += cand[j] > k;
            if (above < a.top) {
                a.top_lp[static_cast<long>(row) * a.top + above] = lp(order_value(static_cast<uint32_t>(k >> 32)));
                a.top_id[static_cast<long>(row) * a.top + above] = static_cast<long>(~static_cast<uint32_t>(k));
            }
        }
    }
    if (parts > 1) cluster_sync();        // the parts' shared memory has been read
}

}  // namespace mica
