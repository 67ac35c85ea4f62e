// Quantize-and-append of packed prompts into the int8 arena.
//
// Per (token, head) row of K and of V, as every other writer of the arena:
//   s = max(max|x| / 127, 1e-12)            IEEE f32 division
//   q = clamp(round_half_even(x / s), -127, 127)
// This file is compiled with -fmad=false -prec-div=true, as quant.cu.
#include "common.cuh"
#include "../host/internal.h"

namespace pp {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxChunk = 64;  // tokens of a CTA

struct AppendArgs {
    const void* src[2];  // K, V
    uint64_t ts[2], hs[2];
    uint8_t* codes[2];
    float* scales[2];
    const uint32_t* starts;
    const uint32_t* offsets;
    uint32_t tokens, branches, heads, capacity, chunk;
    uint32_t vec;
    uint32_t* status;
};

// A lane holds 8 consecutive elements of a row, D / 8 lanes a row.
template <bool BF>
__device__ __forceinline__ void load_row8(const void* p, uint64_t i, bool vec, float (&v)[8]) {
    if constexpr (BF) {
        const uint16_t* s = reinterpret_cast<const uint16_t*>(p) + i;
        if (vec) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(s));
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[2 * k] = bf16_lo_to_f32(w[k]);
                v[2 * k + 1] = bf16_hi_to_f32(w[k]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = bf16_lo_to_f32(s[k]);
        }
    } else {
        const float* s = reinterpret_cast<const float*>(p) + i;
        if (vec) {
            const float4 x = __ldg(reinterpret_cast<const float4*>(s)), y = __ldg(reinterpret_cast<const float4*>(s) + 1);
            v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
            v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = s[k];
        }
    }
}

// CTA x takes `chunk` tokens of all heads, K and V.
template <int D, bool BF>
__global__ void __launch_bounds__(kThreads) prompt_append_kernel(const AppendArgs a) {
    constexpr int L = D / 8;  // lanes of a row
    __shared__ uint64_t dst[kMaxChunk];  // slot of head 0 of each token, or ~0
    const uint32_t t0 = blockIdx.x * a.chunk, n_tok = min(a.chunk, a.tokens - t0);
    pdl_wait_primary();
    int bad = 0;
    for (uint32_t b = threadIdx.x; b < a.branches; b += kThreads)
        bad |= a.starts[b + 1] < a.starts[b] || a.starts[b + 1] > a.tokens;
    if (__syncthreads_or(bad)) {
        if (blockIdx.x == 0 && threadIdx.x == 0 && a.status) atomicOr(a.status, PP_DEV_LENGTH_RANGE);
        return;
    }
    if (threadIdx.x < n_tok) {
        const uint32_t t = t0 + threadIdx.x;
        uint32_t lo = 0, hi = a.branches;  // the last branch that starts at or before t
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (a.starts[mid] <= t) lo = mid;
            else hi = mid;
        }
        uint64_t d = ~0ull;
        if (a.starts[lo] <= t && t < a.starts[lo + 1]) {
            const uint64_t slot = (uint64_t)a.offsets[lo] + (t - a.starts[lo]);
            if (slot < a.capacity) d = (uint64_t)lo * a.heads * a.capacity + slot;
            else if (a.status) atomicOr(a.status, PP_DEV_OFFSET_RANGE);
        }
        dst[threadIdx.x] = d;
    }
    __syncthreads();
    const uint32_t rows = 2 * n_tok * a.heads;
    const int lane = threadIdx.x % L;
    bool finite = true;
    for (uint32_t r = threadIdx.x / L; r < (rows + kThreads / L - 1) / (kThreads / L) * (kThreads / L); r += kThreads / L) {
        const bool in = r < rows;
        const uint32_t kv = in ? r / (n_tok * a.heads) : 0u, i = in ? r - kv * n_tok * a.heads : 0u;
        const uint32_t tok = i / a.heads, head = i - tok * a.heads;
        const uint64_t base = dst[tok];
        const bool on = in && base != ~0ull;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = 0.f;
        if (on) load_row8<BF>(a.src[kv], (uint64_t)(t0 + tok) * a.ts[kv] + head * a.hs[kv] + 8 * lane, a.vec, v);
        float m = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            finite = finite && isfinite(v[k]);
            m = fmaxf(m, fabsf(v[k]));
        }
#pragma unroll
        for (int o = L / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float s = fmaxf(__fdiv_rn(m, 127.f), 1e-12f);
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int q = max(-127, min(127, __float2int_rn(__fdiv_rn(v[k], s))));
            w[k / 4] |= (uint32_t)(q & 0xff) << (8 * (k % 4));
        }
        if (on) {
            const uint64_t slot = base + (uint64_t)head * a.capacity;
            *reinterpret_cast<uint2*>(a.codes[kv] + slot * D + 8 * lane) = make_uint2(w[0], w[1]);
            if (lane == 0) a.scales[kv][slot] = s;
        }
    }
    if (!finite && a.status) atomicOr(a.status, PP_DEV_NONFINITE_INPUT);
}

}  // namespace

cudaError_t launch_prompt_append(const PromptAppendLaunch& P, cudaStream_t stream) {
    AppendArgs a{};
    a.src[0] = P.k;
    a.src[1] = P.v;
    a.ts[0] = P.k_ts;
    a.ts[1] = P.v_ts;
    a.hs[0] = P.k_hs;
    a.hs[1] = P.v_hs;
    a.codes[0] = P.arena->k;
    a.codes[1] = P.arena->v;
    a.scales[0] = P.arena->k_scale;
    a.scales[1] = P.arena->v_scale;
    a.starts = P.starts;
    a.offsets = P.offsets;
    a.tokens = P.tokens;
    a.branches = P.arena->rows / P.arena->heads;
    a.heads = P.arena->heads;
    a.capacity = P.arena->capacity;
    a.vec = P.vec;
    a.status = P.status;
    a.chunk = 4;
    const dim3 grid((P.tokens + a.chunk - 1) / a.chunk);
    if (P.arena->head_dim == 128)
        return P.bf16 ? launch_pdl(prompt_append_kernel<128, true>, grid, dim3(kThreads), stream, a)
                      : launch_pdl(prompt_append_kernel<128, false>, grid, dim3(kThreads), stream, a);
    return P.bf16 ? launch_pdl(prompt_append_kernel<64, true>, grid, dim3(kThreads), stream, a)
                  : launch_pdl(prompt_append_kernel<64, false>, grid, dim3(kThreads), stream, a);
}

}  // namespace pp
