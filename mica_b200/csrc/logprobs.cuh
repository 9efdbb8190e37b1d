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
// with a run of it; a cluster takes row after row. In a CTA one warp keeps bulk copies of the coming
// logits in flight through a ring in shared memory, 20 warps make the pass, and two groups of 4
// warps finish rows in turn while the pass goes on with the next. The parts of a row meet in the first CTA's
// shared memory: one launch, no workspace.
//
// Alternatives without a list in the pass: a thread keeps only the largest logit it has seen. The
// maxima of 64 groups of threads are of disjoint elements, so the top-th largest of them is a lower
// bound of the run's top-th largest logit; only threads whose maximum reaches it can hold an
// alternative (about 25 of 640 for 20 alternatives of random logits), and their vectors are read
// again, from L2, and elements that reach the bound kept. Warps sort them 32 at a time and merge.
//
// Measured (cold L2; in brackets with warm instruction and data caches): 1025 rows of 151936, top 20, bf16 76 us
// (65, 4.8 TB/s), fp16 78 (72), fp32 129 to 138 (118, 5.3 TB/s); 6 rows of 151936 fp32, top 8, 16 us of which 8 are
// a launch. In the bf16 pass the exponential's pipe is busy 63 % of the time, issue 55 %, memory 60 % of its peak:
// none is full, and all three wait at the rows' ends. One CTA a row with a pass for each alternative took 6269 us.
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

constexpr int LP_THREADS = 640;          // make the pass
constexpr int LP_WARPS = LP_THREADS / 32;
constexpr int LP_EPI = 128;              // finish a row; two groups of them take rows in turn
constexpr int LP_BLOCK = LP_THREADS + 32 + 2 * LP_EPI;
constexpr int LP_UNROLL = 4;             // 16-byte vectors of a thread's step
constexpr int LP_STEP = LP_THREADS * LP_UNROLL;         // vectors of a ring stage (40 KB)
constexpr int LP_STAGES = 3;
constexpr int LP_CAND = 512;             // candidates a CTA can rank
constexpr int LP_TOP = 32;
constexpr int LP_BACK = 768;             // vectors read again at once
constexpr int LP_CLUSTER = 16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Logits are held above -2^23 in the sums (2^23 is a bf16 number too), and a row whose maximum is beyond 2^23 or
// not well above -2^23 is computed again without the limit: the pass's weights are 2^fma(z, log2e, -mc), so all of
// them, the largest's too, carry mc's rounding as a factor, which cancels but has to be small; up to |mc| = 2^24
// it is within 2^-0.5 .. 2^0.5. Below the limit a weight is 0 in any row that is not computed again.
constexpr float LP_FLOOR = -8388608.f;

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
    if constexpr (std::is_same<T, float>::value) return v;
    else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
    else return __bfloat162float(v);
}
__device__ __forceinline__ void lp_sync(int g) { named_bar_sync(1 + g, LP_EPI); }   // a group that finishes a row
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
    const float fa = fast_exp2(da), fb = fast_exp2(db);
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

// One thread's step: its sums and largest logit take in U vectors.
template <typename T, int U>
__device__ __forceinline__ void lp_step(const uint4 (&q)[U], LpSums& a, float& top) {
    constexpr int N = LpVec<T>::N;
    float cm;
    uint4 c[U];
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {       // maxima of pairs
        __nv_bfloat162 m2 = *reinterpret_cast<const __nv_bfloat162*>(&q[0].x);
        const __nv_bfloat162 lo2 = __float2bfloat162_rn(LP_FLOOR);
#pragma unroll
        for (int u = 0; u < U; ++u) {
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
        for (int u = 0; u < U; ++u) {
            LpVec<T>::values(q[u], f);
#pragma unroll
            for (int i = 0; i < N; ++i) cm = max_nan(cm, f[i]);
            c[u] = q[u];
        }
    }
    top = max_nan(top, cm);
    const float cmc = max_nan(cm, LP_FLOOR) * kLog2e;
    if (!(cmc <= a.mc)) {
        const float d = fmaxf(a.mc - cmc, -1000.f), f = fast_exp2(d);
        a.w = f * fmaf(d, a.s, a.w);
        a.s *= f;
        a.mc = cmc;
    }
    const unsigned long long c2 = f2_pack(kLog2e, kLog2e), n2 = f2_pack(-a.mc, -a.mc);
    unsigned long long s2 = 0ull, w2 = 0ull;
#pragma unroll
    for (int u = 0; u < U; ++u) {
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

struct LpPart {                 // what a CTA tells its cluster of a row
    LpSums sums;
    float top;                  // its largest logit as it is
    int count;                  // entries of list, in order
    int pad;
    unsigned long long list[LP_TOP];
};

// The row by the LP_EPI threads, in passes, for maxima near the type's ends, infinities and NaN: the
// definition literally.
__device__ __forceinline__ float lp_reduce(float v, bool max, float* red, int g) {
    v = max ? warp_max(v) : warp_sum(v);
    lp_sync(g);
    if ((threadIdx.x & 31) == 0) red[((threadIdx.x - LP_THREADS - 32) >> 5) & 3] = v;
    lp_sync(g);
    v = red[0];
    for (int i = 1; i < LP_EPI / 32; ++i) v = max ? fmaxf(v, red[i]) : v + red[i];
    return v;
}
template <typename T>
__device__ __noinline__ void lp_row_plain(const LogprobArgs& a, const T* z, int e, int g, float* red, float& m,
                                          float& logs, float& ent) {
    m = -INFINITY;
    float odd = 0.f;
    for (int i = e; i < a.V; i += LP_EPI) {
        const float v = to_f32(z[i]);
        if (v != v || v == INFINITY) odd = 1.f;
        m = fmaxf(m, v);
    }
    odd = lp_reduce(odd, true, red, g);
    m = lp_reduce(m, true, red, g);
    float s = 0.f, w = 0.f;
    for (int i = e; i < a.V; i += LP_EPI) {
        const float d = to_f32(z[i]) - m, x = m == -INFINITY ? 0.f : expf(d);
        s += x;
        if (x > 0.f) w -= d * x;
    }
    s = lp_reduce(s, false, red, g);
    w = lp_reduce(w, false, red, g);
    logs = m == -INFINITY ? 0.f : logf(s);
    ent = m == -INFINITY ? 0.f : logs + w / s;
    if (odd > 0.f) logs = ent = nan_f32();
}

// The largest `top` keys of elements [i0, i1), each by one pass: for runs with more large values in a
// few threads than a list holds.
template <typename T>
__device__ __noinline__ void lp_select_plain(const T* z, int i0, int i1, int e, int g, int top, unsigned long long* list,
                                             unsigned long long* best) {
    unsigned long long last = ~0ull;
    for (int j = 0; j < top; ++j) {
        unsigned long long b = 0ull;
        for (int i = i0 + e; i < i1; i += LP_EPI) {
            const unsigned long long c = rank_key(to_f32(z[i]), i);
            if (c < last && c > b) b = c;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long c = __shfl_xor_sync(0xffffffffu, b, o);
            b = c > b ? c : b;
        }
        lp_sync(g);
        if ((e & 31) == 0) best[e >> 5] = b;
        lp_sync(g);
        for (int i = 0; i < LP_EPI / 32; ++i) b = best[i] > b ? best[i] : b;
        last = b;
        if (e == 0) list[j] = b;
    }
    lp_sync(g);
}

// Sorts 32 keys across the lanes, largest first.
__device__ __noinline__ unsigned long long lp_sort32(unsigned long long k, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, k, o);
            const bool down = (lane & size) == 0 || size == 32;      // this run: largest first
            const bool low = (lane & o) == 0;
            if ((k < other) == (low == down)) k = other;
        }
    return k;
}
// The 32 largest of two sorted sets, sorted.
__device__ __noinline__ unsigned long long lp_merge32(unsigned long long a, unsigned long long b, int lane) {
    const unsigned long long r = __shfl_sync(0xffffffffu, b, 31 - lane);
    unsigned long long k = a > r ? a : r;                            // bitonic
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, k, o);
        if ((k < other) == ((lane & o) == 0)) k = other;
    }
    return k;
}

// Joins the lanes' sums: the maximum first, then each is rescaled to it once and added, in a fixed
// order; every lane gets the same bits. (Not inlined, as the sort and the merge: a row is finished once
// in thousands of instructions of the pass, so its code is fetched anew, and that took longer than
// running it.)
__device__ __noinline__ LpSums lp_join_warp(LpSums a) {
    float mc = a.mc;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mc = max_nan(mc, __shfl_xor_sync(0xffffffffu, mc, o));
    const float d = fmaxf(a.mc - mc, -1000.f), f = fast_exp2(d);
    float s = a.s * f, w = f * fmaf(d, a.s, a.w);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        w += __shfl_xor_sync(0xffffffffu, w, o);
    }
    return LpSums{mc, s, w};
}

__device__ __forceinline__ void st_cluster(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, unsigned long long v) {
    asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
// Bounded wait on a barrier that CTAs of the cluster arrive on.
__device__ __forceinline__ bool lp_wait_cluster(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag) {
    const unsigned long long t0 = global_ns();
    for (;;) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
        if (ok) return true;
        if (*abort_flag) return false;
        if (global_ns() - t0 > kWaitLimitNs) {
            *abort_flag = 1u;
            atomicExch(&g_dev_error, MICA_DEV_TIMEOUT_GRID);
            return false;
        }
    }
}

// A row's 16-byte vectors and the single elements before and behind them, and CTA `rank`'s part.
template <typename T>
struct LpRow {
    const T* z;
    int head, nvec, v0, v1;
    __device__ __forceinline__ LpRow(const LogprobArgs& a, int row, int rank, int parts) {
        z = static_cast<const T*>(a.z) + static_cast<long>(row) * a.ld;
        head = min(a.V, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / static_cast<int>(sizeof(T)));
        nvec = (a.V - head) / LpVec<T>::N;
        v0 = static_cast<int>(static_cast<long>(nvec) * rank / parts);
        v1 = static_cast<int>(static_cast<long>(nvec) * (rank + 1) / parts);
    }
    __device__ __forceinline__ const uint4* vectors() const { return reinterpret_cast<const uint4*>(z + head); }
    // thread t's single element, -1 for none: fewer than 8 at either end, the first and the last CTA's
    __device__ __forceinline__ int single(const LogprobArgs& a, int t, int rank, int parts) const {
        const int tail = head + nvec * LpVec<T>::N;
        return rank == 0 && t < head                                   ? t
               : rank == parts - 1 && t >= 16 && tail + (t - 16) < a.V ? tail + (t - 16) : -1;
    }
};

struct LpGroup {                // what finishing a row works on
    unsigned long long cand[LP_CAND];
    unsigned long long list[4][LP_TOP];
    uint4 back[LP_BACK];                 // vectors read again
    int back_at[LP_BACK], hit[LP_BACK];
    int who[LP_THREADS];
    uint32_t group[64], bound;           // order keys
    float red[4], top[4];
    LpSums sums[4];
    int count, n_who, n_hit;
};
struct LpShared {
    float4 mine[2][LP_THREADS];          // of each thread of the pass: sums and largest logit, rows in turn
    LpPart slots[2][LP_CLUSTER];         // of the first CTA: the parts of a row, rows in turn
    LpGroup work[2];
    uint64_t full[LP_STAGES], empty[LP_STAGES], passed[2], done[2], ready[2], taken[2];
    uint32_t abort;
};
constexpr int LP_SMEM = 128 + LP_STAGES * LP_STEP * 16 + static_cast<int>(sizeof(LpShared));
static_assert(LP_SMEM <= 232448, "shared memory of a CTA");

template <typename T>
__global__ void __launch_bounds__(LP_BLOCK, 1) token_logprobs_kernel(const LogprobArgs a, const int parts) {
    constexpr int N = LpVec<T>::N;
    extern __shared__ __align__(128) uint4 ring[];
    LpShared& sh = *reinterpret_cast<LpShared*>(ring + LP_STAGES * LP_STEP);
    volatile uint32_t* abort_flag = &sh.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = parts > 1 ? static_cast<int>(cluster_ctarank()) : 0;
    const int first_row = blockIdx.x / parts, rows_step = gridDim.x / parts;
    if (threadIdx.x == 0) {
        for (int i = 0; i < LP_STAGES; ++i) {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.empty[i], LP_WARPS);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.passed[i], LP_WARPS);
            mbar_init(&sh.done[i], 1);
            mbar_init(&sh.ready[i], parts);
            mbar_init(&sh.taken[i], 1);
        }
        sh.abort = 0u;
        fence_mbar_init();
    }
    if (parts > 1) cluster_sync(); else __syncthreads();

    // A wait that gives up lets the loops run on over whatever is there; the error word says so.
    if (warp == LP_WARPS) {
        // ---------------------------------- loads ----------------------------------
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            for (int row = first_row; row < a.N && ok; row += rows_step) {
                const LpRow<T> r(a, row, rank, parts);
                for (int v = r.v0; v < r.v1; v += LP_STEP, ++it) {
                    const int st = it % LP_STAGES;
                    ok = mbar_wait(&sh.empty[st], ((it / LP_STAGES) & 1u) ^ 1u, abort_flag, MICA_DEV_TIMEOUT_PRODUCER);
                    if (!ok) break;
                    const uint32_t bytes = min(LP_STEP, r.v1 - v) * 16;
                    mbar_arrive_expect_tx(&sh.full[st], bytes);
                    asm volatile(
                        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                        ::"r"(smem_u32(ring + st * LP_STEP)), "l"(reinterpret_cast<uint64_t>(r.vectors() + v)), "r"(bytes),
                        "r"(smem_u32(&sh.full[st])) : "memory");
                }
            }
            // copies in flight land before shared memory is released
            for (int i = it > LP_STAGES ? it - LP_STAGES : 0; i < it; ++i)
                mbar_wait(&sh.full[i % LP_STAGES], (i / LP_STAGES) & 1u, abort_flag, MICA_DEV_TIMEOUT_DRAIN);
        }
        __syncwarp();
    } else if (warp < LP_WARPS) {
        // ---------------------------------- the pass ----------------------------------
        constexpr uint32_t kNone = std::is_same<T, float>::value ? 0xff800000u
                                   : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;    // -inf
        int it = 0, nth = 0;
        const int tid = threadIdx.x;
        for (int row = first_row; row < a.N; row += rows_step, ++nth) {
            const LpRow<T> r(a, row, rank, parts);
            const int my_single = r.single(a, tid, rank, parts);
            const float single = my_single >= 0 ? to_f32(r.z[my_single]) : 0.f;
            LpSums sums{LP_FLOOR * kLog2e, 0.f, 0.f};
            float top = -INFINITY;
            for (int v = r.v0; v < r.v1; v += LP_STEP, ++it) {
                const int st = it % LP_STAGES;
                const uint4* in = ring + st * LP_STEP + tid;
                mbar_wait(&sh.full[st], (it / LP_STAGES) & 1u, abort_flag, MICA_DEV_TIMEOUT_EPILOGUE);
                if (v + LP_STEP <= r.v1) {
                    uint4 q[LP_UNROLL];
#pragma unroll
                    for (int u = 0; u < LP_UNROLL; ++u) q[u] = in[u * LP_THREADS];
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.empty[st]);
                    lp_step<T>(q, sums, top);
                } else {
                    // the row's last stage: a vector at a time
                    for (int u = v + warp * 32; u < r.v1; u += LP_THREADS, in += LP_THREADS) {
                        uint4 q[1] = {u + lane < r.v1 ? *in : make_uint4(kNone, kNone, kNone, kNone)};
                        lp_step<T>(q, sums, top);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.empty[st]);
                }
            }
            if (my_single >= 0) {
                top = max_nan(top, single);
                // with the rounding of mc in its weight, as every other element's
                const float z = max_nan(single, LP_FLOOR), mc = z * kLog2e, d = fmaf(z, kLog2e, -mc), x = fast_exp2(d);
                sums = lp_join(sums, LpSums{mc, x, d * x});
            }
            const int slot = nth & 1;
            if (nth >= 2) mbar_wait(&sh.done[slot], ((nth >> 1) - 1) & 1u, abort_flag, MICA_DEV_TIMEOUT_EPILOGUE);
            sh.mine[slot][tid] = make_float4(sums.mc, sums.s, sums.w, top);
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.passed[slot]);
        }
    } else {
        // ---------------------------------- finishing rows ----------------------------------
        const int g = (warp - LP_WARPS - 1) / (LP_EPI / 32);
        const int e = (threadIdx.x - LP_THREADS - 32) % LP_EPI, ew = e >> 5, slot = g;
        LpGroup& wk = sh.work[g];
        int nth = g;
        for (long next = first_row + static_cast<long>(g) * rows_step; next < a.N; next += 2l * rows_step, nth += 2) {
            const int row = static_cast<int>(next);
            const LpRow<T> r(a, row, rank, parts);
            const uint32_t turn = (nth >> 1) & 1u;
            if (e == 0) wk.count = wk.n_who = 0;
            // the given tokens are on their way during the pass
            long id = -1;
            if (rank == 0 && e < a.M) id = a.ids[static_cast<long>(row) * a.ld_ids + e];
            mbar_wait(&sh.passed[slot], turn, abort_flag, MICA_DEV_TIMEOUT_EPILOGUE);
            // five threads' sums and maxima each; two of these are a group
            constexpr int kEach = LP_THREADS / LP_EPI;
            LpSums sums;
            float4 five[kEach];
            float top = -INFINITY, mc = -INFINITY;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                five[i] = sh.mine[slot][e + i * LP_EPI];
                top = max_nan(top, five[i].w);
                mc = max_nan(mc, five[i].x);
            }
            sums = LpSums{mc, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const float d = fmaxf(five[i].x - mc, -1000.f), f = fast_exp2(d);
                sums.s = fmaf(five[i].y, f, sums.s);
                sums.w = fmaf(f, fmaf(d, five[i].y, five[i].z), sums.w);
            }
            sums = lp_join_warp(sums);
            if (lane == 0) wk.sums[ew] = sums;
            const float pair = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
            if ((e & 1) == 0) wk.group[e >> 1] = order_key(pair);
#pragma unroll
            for (int o = 16; o > 1; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
            top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
            if (lane == 0) wk.top[ew] = top;
            lp_sync(g);
            unsigned long long best = 0ull;          // of warp 0: the run's alternatives in order
            int n = 0;
            if (a.top > 0) {
                {
                    // the top-th largest of the 64 maxima; two threads count for each
                    const int i0 = e >> 1;
                    const uint32_t me = wk.group[i0];
                    int above = 0;
                    const uint4* g4 = reinterpret_cast<const uint4*>(wk.group) + (e & 1) * 8;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint4 k = g4[i];
                        const int at = (e & 1) * 32 + i * 4;
                        above += (k.x > me || (k.x == me && at < i0)) + (k.y > me || (k.y == me && at + 1 < i0)) +
                                 (k.z > me || (k.z == me && at + 2 < i0)) + (k.w > me || (k.w == me && at + 3 < i0));
                    }
                    above += __shfl_xor_sync(0xffffffffu, above, 1);
                    if (above == a.top - 1 && (e & 1) == 0) wk.bound = me;
                }
                lp_sync(g);
                const uint32_t bkey = wk.bound;
                const int n_mine = r.v1 - r.v0, per = (n_mine + LP_THREADS - 1) / LP_THREADS;
                // threads of the pass whose maximum reaches the bound, then their vectors' elements that do
                // (strict: are above it)
#pragma unroll
                for (int i = 0; i < kEach; ++i)
                    if (order_key(five[i].w) >= bkey) wk.who[atomicAdd(&wk.n_who, 1)] = e + i * LP_EPI;
                const auto gather = [&](bool strict) {
                    const auto keep = [&](float f, int id) {
                        const uint32_t k = order_key(f);
                        if (strict ? k > bkey : k >= bkey) {
                            const int at = atomicAdd(&wk.count, 1);
                            if (at < LP_CAND) wk.cand[at] = rank_key(f, id);
                        }
                    };
                    // their vectors come into shared memory, LP_BACK at a time; of those with an element that
                    // passes, each element is a thread's
                    const int items = wk.n_who * per;
                    for (int b0 = 0; b0 < items; b0 += LP_BACK) {
                        const int nb = min(LP_BACK, items - b0);
#pragma unroll 1
                        for (int i = e; i < nb; i += LP_EPI) {
                            const int w = (b0 + i) / per, at = wk.who[w] + (b0 + i - w * per) * LP_THREADS;
                            wk.back_at[i] = at;
                            if (at < n_mine)
                                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(&wk.back[i])),
                                             "l"(reinterpret_cast<uint64_t>(r.vectors() + r.v0 + at)) : "memory");
                        }
                        if (e == 0) wk.n_hit = 0;
                        asm volatile("cp.async.wait_all;" ::: "memory");
                        lp_sync(g);
#pragma unroll 1
                        for (int i = e; i < nb; i += LP_EPI) {
                            if (wk.back_at[i] >= n_mine) continue;
                            float f[N];
                            LpVec<T>::values(wk.back[i], f);
#pragma unroll
                            for (int k = 1; k < N; ++k) f[0] = max_nan(f[0], f[k]);
                            if (order_key(f[0]) >= bkey) wk.hit[atomicAdd(&wk.n_hit, 1)] = i;
                        }
                        lp_sync(g);
                        const int nh = wk.n_hit * N;
#pragma unroll 1
                        for (int i = e; i < nh; i += LP_EPI) {
                            const int b = wk.hit[i / N];
                            keep(to_f32(reinterpret_cast<const T*>(&wk.back[b])[i % N]),
                                 r.head + (r.v0 + wk.back_at[b]) * N + i % N);
                        }
                        if (b0 + LP_BACK < items) lp_sync(g);
                    }
                    const int my_single = r.single(a, e, rank, parts);
                    if (my_single >= 0) keep(to_f32(r.z[my_single]), my_single);
                };
                lp_sync(g);
                gather(false);
                lp_sync(g);
                n = wk.count;
                // the run's elements
                const int lo = rank == 0 ? 0 : r.head + r.v0 * N, hi = rank == parts - 1 ? a.V : r.head + r.v1 * N;
                bool plain = false;
                if (n > LP_CAND) {
                    // more ties at the bound than places (a row that allows few tokens, or equal logits): those
                    // above it, then the first ones at it in order of their ids
                    lp_sync(g);
                    if (e == 0) wk.count = 0;
                    lp_sync(g);
                    gather(true);
                    lp_sync(g);
                    n = wk.count;
                    plain = n > LP_CAND - LP_TOP;
                    const int want = plain ? 0 : n + a.top;              // enough of them
                    for (int i0 = lo; i0 < hi && n < want; i0 += LP_EPI) {
                        const int i = i0 + e;
                        const bool hit = i < hi && order_key(to_f32(r.z[i])) == bkey;
                        const uint32_t bits = __ballot_sync(0xffffffffu, hit);
                        lp_sync(g);
                        if (lane == 0) wk.red[ew] = __int_as_float(__popc(bits));
                        lp_sync(g);
                        int at = n;
                        for (int w = 0; w < LP_EPI / 32; ++w) {
                            const int k = __float_as_int(wk.red[w]);
                            if (w < ew) at += k;
                            n += k;
                        }
                        at += __popc(bits & ((1u << lane) - 1u));
                        if (hit && at < want) wk.cand[at] = rank_key(order_value(bkey), i);
                        n = min(n, want);
                    }
                    lp_sync(g);
                }
                if (plain) {
                    lp_select_plain(r.z, lo, hi, e, g, a.top, wk.list[0], wk.cand);
                    n = min(a.top, hi - lo);
                    best = lane < n ? wk.list[0][lane] : 0ull;
                } else {
                    // each warp sorts 32 at a time and keeps the 32 largest
                    for (int i = ew * 32; i < n; i += LP_EPI) {
                        const unsigned long long k = lp_sort32(i + lane < n ? wk.cand[i + lane] : 0ull, lane);
                        best = i == ew * 32 ? k : lp_merge32(best, k, lane);
                    }
                    if (n > 32) {
                        wk.list[ew][lane] = best;
                        lp_sync(g);
                        if (ew == 0)
                            for (int w = 1; w < LP_EPI / 32; ++w) best = lp_merge32(best, wk.list[w][lane], lane);
                    }
                    n = min(n, a.top);
                }
            }

            float given = rank == 0 && id >= 0 && id < a.V ? to_f32(r.z[id]) : 0.f;

            // ---- to the first CTA ----
            if (ew == 0) {
                if (lane == 0) mbar_arrive(&sh.done[slot]);
                float top_all = max_nan(max_nan(wk.top[0], wk.top[1]), max_nan(wk.top[2], wk.top[3]));
                sums = lp_join_warp(lane < 4 ? wk.sums[lane] : LpSums{LP_FLOOR * kLog2e, 0.f, 0.f});
                // the slot's last row has been taken
                if (parts > 1 && nth >= 2) lp_wait_cluster(&sh.taken[slot], turn ^ 1u, abort_flag);
                const uint32_t here = smem_u32(&sh.slots[slot][rank]), to = parts > 1 ? map_to_rank(here, 0) : here;
                if (lane < n) st_cluster(to + offsetof(LpPart, list) + lane * 8, best);
                if (lane == 0) {
                    st_cluster(to, sums.mc);
                    st_cluster(to + 4, sums.s);
                    st_cluster(to + 8, sums.w);
                    st_cluster(to + offsetof(LpPart, top), top_all);
                    st_cluster(to + offsetof(LpPart, count), __int_as_float(n));
                }
                __syncwarp();
                if (lane == 0) {
                    if (parts > 1) {
                        asm volatile("fence.acq_rel.cluster;" ::: "memory");
                        mbar_arrive_cluster(map_to_rank(smem_u32(&sh.ready[slot]), 0));
                    } else {
                        mbar_arrive(&sh.ready[slot]);
                    }
                }
            }
            if (rank != 0) { lp_sync(g); continue; }

            // ---- the row ----
            lp_wait_cluster(&sh.ready[slot], turn, abort_flag);
            const LpPart* p = sh.slots[slot];
            sums = p[0].sums;
            if (parts > 1) sums = lp_join_warp(lane < parts ? p[lane].sums : LpSums{LP_FLOOR * kLog2e, 0.f, 0.f});
            float top_all = lane < parts ? p[lane].top : -INFINITY;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) top_all = max_nan(top_all, __shfl_xor_sync(0xffffffffu, top_all, o));
            top_all = __shfl_sync(0xffffffffu, top_all, 0);
            if (a.top > 0) {
                // warp w merges the lists of parts w, w + 4, ..., warp 0 the four results
                best = 0ull;
                for (int i = ew; i < parts; i += LP_EPI / 32) {
                    const unsigned long long k = lane < p[i].count ? p[i].list[lane] : 0ull;
                    best = i == ew ? k : lp_merge32(best, k, lane);
                }
                if (parts > 1) {
                    wk.list[ew][lane] = best;
                    lp_sync(g);
                    if (ew == 0)
                        for (int w = 1; w < min(parts, LP_EPI / 32); ++w) best = lp_merge32(best, wk.list[w][lane], lane);
                }
            }
            // where the sums are those of the largest logit alone, to the bit, its log probability and the entropy are
            // zero, not the difference of two roundings
            const float d_top = fmaf(top_all, kLog2e, -sums.mc), x_top = fast_exp2(d_top);
            const bool alone = sums.s == x_top && sums.w == d_top * x_top;
            const float log2s = alone ? d_top : log2f(sums.s);
            float m = -INFINITY, logs = 0.f, ent = kLn2 * (log2s - sums.w / sums.s);
            // nothing allowed; or beyond the range of the sums, or NaN
            const bool none = top_all == -INFINITY;
            const bool odd = !none && !(sums.mc > 0.1f * LP_FLOOR && sums.mc < -LP_FLOOR && sums.s > 0.f && sums.s < INFINITY);
            if (none || alone) ent = 0.f;
            if (odd) lp_row_plain(a, r.z, e, g, wk.red, m, logs, ent);
            const auto lp = [&](float f) {
                if (none) return -INFINITY;
                if (odd) return (f - m) - logs;
                if (f < 8.f * LP_FLOOR) return f - (sums.mc + log2s) * kLn2;       // f * log2e may pass fp32's range
                return (fmaf(f, kLog2e, -sums.mc) - log2s) * kLn2;
            };
            if (e == 0) a.entropy[row] = ent;
            for (int j = e; j < a.M; j += LP_EPI) {
                if (j != e) {
                    id = a.ids[static_cast<long>(row) * a.ld_ids + j];
                    given = id >= 0 && id < a.V ? to_f32(r.z[id]) : 0.f;
                }
                a.logprob[static_cast<long>(row) * a.M + j] = id < 0 ? 0.f : id >= a.V ? nan_f32() : lp(given);
            }
            if (ew == 0 && lane < a.top) {
                a.top_lp[static_cast<long>(row) * a.top + lane] = lp(order_value(static_cast<uint32_t>(best >> 32)));
                a.top_id[static_cast<long>(row) * a.top + lane] = static_cast<long>(~static_cast<uint32_t>(best));
            }
            lp_sync(g);                            // the slot has been read
            if (parts > 1 && e < parts) mbar_arrive_cluster(map_to_rank(smem_u32(&sh.taken[slot]), e));
        }
    }
    if (parts > 1) cluster_sync();        // no CTA ends while another may still write to it
}

}  // namespace mica
