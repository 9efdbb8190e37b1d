// logprobs.cuh -- log probabilities of given tokens, entropy and top alternatives of logits rows.
//
//   m = max_v z_v,  S = sum_v e^(z_v - m),  lse = m + log S
//   logprob[r, j] = z[r, ids[r, j]] - lse        (a negative id is padding: 0; one past the end: NaN)
//   entropy[r]    = log S + sum_v (m - z_v) e^(z_v - m) / S          (a sum of terms >= 0)
//   top[r, j]     = the j-th largest z - lse and its id, ties to the lowest id, NaN before all
// A row whose logits are all -inf allows nothing: log probabilities -inf, entropy 0.
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

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
    if constexpr (std::is_same<T, float>::value) return v;
    else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
    else return __bfloat162float(v);
}

// Orders logits for the alternatives: larger value first, NaN above +inf, -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float z) {
    if (z != z) return 0xffffffffu;
    const uint32_t u = __float_as_uint(z + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t k) {
    if (k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// Simplest form: one block per row, one pass for the maximum, one for the sums, one for each
// alternative.
template <typename T>
__global__ void __launch_bounds__(512) token_logprobs_kernel(const LogprobArgs a) {
    __shared__ float red[32];
    __shared__ unsigned long long best[16];
    const int row = blockIdx.x;
    const T* z = static_cast<const T*>(a.z) + static_cast<long>(row) * a.ld;
    float m = -INFINITY;
    bool nan = false;
    for (int i = threadIdx.x; i < a.V; i += blockDim.x) {
        const float v = to_f32(z[i]);
        nan |= v != v;
        m = fmaxf(m, v);
    }
    nan = __syncthreads_or(nan);
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int i = 0; i < (blockDim.x >> 5); ++i) m = fmaxf(m, red[i]);
    __syncthreads();
    float s = 0.f, w = 0.f;
    for (int i = threadIdx.x; i < a.V; i += blockDim.x) {
        const float d = to_f32(z[i]) - m, e = m == -INFINITY ? 0.f : expf(d);
        s += e;
        if (e > 0.f) w -= d * e;
    }
    s = block_reduce<false>(s, red);
    __syncthreads();
    w = block_reduce<false>(w, red);
    float logs = logf(s);
    float ent = logs + w / s;
    if (m == -INFINITY) { logs = 0.f; ent = 0.f; }
    if (nan) logs = ent = __uint_as_float(0x7fc00000u);
    const auto lp = [&](float v) { return m == -INFINITY && !nan ? -INFINITY : (v - m) - logs; };
    if (threadIdx.x == 0) a.entropy[row] = ent;
    for (int j = threadIdx.x; j < a.M; j += blockDim.x) {
        const long id = a.ids[static_cast<long>(row) * a.ld_ids + j];
        a.logprob[static_cast<long>(row) * a.M + j] =
            id < 0 ? 0.f : id >= a.V ? __uint_as_float(0x7fc00000u) : lp(to_f32(z[id]));
    }
    unsigned long long last = ~0ull;      // (key << 32) | ~id of the alternative before
    for (int j = 0; j < a.top; ++j) {
        unsigned long long b = 0ull;
        for (int i = threadIdx.x; i < a.V; i += blockDim.x) {
            const unsigned long long c = static_cast<unsigned long long>(order_key(to_f32(z[i]))) << 32 | ~static_cast<uint32_t>(i);
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
        for (int i = 0; i < (blockDim.x >> 5); ++i) b = best[i] > b ? best[i] : b;
        last = b;
        if (threadIdx.x == 0) {
            a.top_lp[static_cast<long>(row) * a.top + j] = lp(order_value(static_cast<uint32_t>(b >> 32)));
            a.top_id[static_cast<long>(row) * a.top + j] = static_cast<long>(~static_cast<uint32_t>(b));
        }
    }
}

}  // namespace mica
