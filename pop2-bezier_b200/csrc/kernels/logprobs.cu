// Log probabilities of given tokens, entropy, rank and the best alternatives
// of rows of logits.
//
// With m the largest logit of the window and e_i = exp(x_i - m), one pass
// keeps (m, s, d): s = sum of e_i without the largest itself, d = sum of
// e_i (m - x_i).  Then
//   log p_t = (x_t - m) - log1p(s)         entropy = log1p(s) + d / (1 + s)
// Leaving the largest out of s keeps what is left of a nearly certain token's
// log probability, which 1 + s would round away, and both terms of the entropy
// are positive, so nothing cancels.  When the running maximum rises by g, s
// becomes (s + 1) exp(-g) and d becomes (d + g (s + 1)) exp(-g).
#include <math_constants.h>

#include "common.cuh"
#include "../host/internal.h"

namespace pp {
namespace {

constexpr int kThreads = 256;

struct Args {
    const void* logits;
    uint64_t stride;
    const int32_t* targets;
    const uint32_t* bounds;
    uint32_t rows, choices, top;
    float* logprob;
    float* entropy;
    uint32_t* rank;
    uint32_t* top_ids;
    float* top_logprobs;
    uint32_t* status;
};

struct Mass {
    float m, s, d;
};

__device__ __forceinline__ Mass merge(Mass a, Mass b) {
    if (b.m > a.m) {
        const Mass t = a;
        a = b;
        b = t;
    }
    if (b.m == -CUDART_INF_F) return a;  // nothing in b (or nothing but -inf)
    const float g = a.m - b.m, f = expf(-g);
    if (f > 0.f) {  // g may be inf between the types' ends
        a.d += (b.d + g * (b.s + 1.f)) * f;
        a.s += (b.s + 1.f) * f;
    }
    return a;
}

// Order of the alternatives: larger logit first, then lower column.  -0 and +0
// are one value; NaN lies below -inf.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0u;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t kKeyNegInf = 0x007fffffu;  // order_key(-inf)

__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

template <bool BF>
__device__ __forceinline__ float load_logit(const void* p, uint64_t i) {
    if constexpr (BF) return bf16_lo_to_f32(__ldg(reinterpret_cast<const unsigned short*>(p) + i));
    else return __ldg(reinterpret_cast<const float*>(p) + i);
}

template <bool BF>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const Args a) {
    __shared__ Mass s_mass[kThreads / 32];
    __shared__ uint32_t s_rank, s_nan;
    __shared__ unsigned long long s_best[kThreads / 32], s_prev;
    const uint32_t row = blockIdx.x, t = threadIdx.x;
    pdl_wait_primary();
    if (t == 0) s_rank = s_nan = 0;
    __syncthreads();
    const uint64_t base = (uint64_t)row * a.stride;
    uint32_t lo = 0, n = a.choices;
    if (a.bounds) {
        lo = a.bounds[2 * row];
        n = a.bounds[2 * row + 1];
        if ((uint64_t)lo + n > a.choices) {
            if (t == 0 && a.status) atomicOr(a.status, PP_DEV_WINDOW_RANGE);
            lo = n = 0;
        }
    }
    const int64_t target = a.targets[row];
    const bool inside = target >= lo && target < (int64_t)lo + n;
    const float xt = inside ? load_logit<BF>(a.logits, base + target) : -CUDART_INF_F;
    const uint32_t kt = order_key(xt);
    Mass mass{-CUDART_INF_F, 0.f, 0.f};
    uint32_t ahead = 0;
    bool nan = false;
    for (uint32_t i = t; i < n; i += kThreads) {
        const float x = load_logit<BF>(a.logits, base + lo + i);
        const uint32_t k = order_key(x);
        ahead += !inside || k > kt || (k == kt && lo + i < target);
        nan |= !(x < CUDART_INF_F);
        mass = merge(mass, Mass{x, 0.f, 0.f});
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        mass = merge(mass, Mass{__shfl_xor_sync(0xffffffffu, mass.m, o), __shfl_xor_sync(0xffffffffu, mass.s, o),
                                __shfl_xor_sync(0xffffffffu, mass.d, o)});
        ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
    }
    if ((t & 31) == 0) {
        s_mass[t >> 5] = mass;
        atomicAdd(&s_rank, ahead);
    }
    if (nan) s_nan = 1;
    __syncthreads();
    mass = s_mass[0];
    for (int w = 1; w < kThreads / 32; ++w) mass = merge(mass, s_mass[w]);
    const bool void_row = s_nan || mass.m == -CUDART_INF_F;
    const double lse1 = log1p((double)mass.s);  // log of the sum, less m
    if (t == 0) {
        a.logprob[row] = void_row ? CUDART_NAN_F : (float)((double)xt - (double)mass.m - lse1);
        a.entropy[row] = void_row ? CUDART_NAN_F : (float)(lse1 + (double)mass.d / (1.0 + (double)mass.s));
        a.rank[row] = s_rank;
        s_prev = ~0ull;
    }
    for (uint32_t j = 0; j < a.top; ++j) {
        __syncthreads();
        unsigned long long best = 0;
        const unsigned long long prev = s_prev;
        for (uint32_t i = t; i < n; i += kThreads) {
            const unsigned long long k =
                (unsigned long long)order_key(load_logit<BF>(a.logits, base + lo + i)) << 32 | ~(lo + i);
            if (k < prev && k > best) best = k;
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if ((t & 31) == 0) s_best[t >> 5] = best;
        __syncthreads();
        if (t == 0) {
            for (int w = 1; w < kThreads / 32; ++w) best = max(best, s_best[w]);
            const bool some = (uint32_t)(best >> 32) > kKeyNegInf;
            a.top_ids[(uint64_t)row * a.top + j] = some ? ~(uint32_t)best : 0xffffffffu;
            float lp = -CUDART_INF_F;
            if (some) lp = void_row ? CUDART_NAN_F : (float)((double)key_value((uint32_t)(best >> 32)) - (double)mass.m - lse1);
            a.top_logprobs[(uint64_t)row * a.top + j] = lp;
            s_prev = best;
        }
    }
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobsLaunch& L, cudaStream_t stream) {
    Args a{};
    a.logits = L.logits;
    a.stride = L.row_stride;
    a.targets = L.targets;
    a.bounds = L.bounds;
    a.rows = L.rows;
    a.choices = L.choices;
    a.top = L.top;
    a.logprob = L.logprob;
    a.entropy = L.entropy;
    a.rank = L.rank;
    a.top_ids = L.top_ids;
    a.top_logprobs = L.top_logprobs;
    a.status = L.status;
    return L.bf16 ? launch_pdl(logprobs_kernel<true>, dim3(L.rows), dim3(kThreads), stream, a)
                  : launch_pdl(logprobs_kernel<false>, dim3(L.rows), dim3(kThreads), stream, a);
}

}  // namespace pp
