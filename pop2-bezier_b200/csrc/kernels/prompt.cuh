// Shared by the prompt attention kernels: the work list in the workspace, and a
// row computed by itself.
//
// A work item is one K/V head of one entry; an entry is 256 consecutive query
// rows of one sequence against a range of its keys.  The G = heads / kv_heads
// query heads that read one K/V head are packed into the rows, so that each
// key tile is loaded once for all of them: tile t (0, 1) of an entry holds
// tpt = floor(128 / G) tokens, its row r token tok0 + t * tpt + r / G and head
// kv_head * G + r % G.  Causal rows of one tile then also see almost the same
// keys.  A row sees `visible` = nk (or nk - nq + token + 1) keys.
#pragma once

#include <stdint.h>

#include "../host/internal.h"
#include "common.cuh"

namespace pp {

constexpr uint32_t kPromptTileRows = 128;  // rows of a tile, two tiles an entry
constexpr uint32_t kPromptKeyTile = 128;   // keys of a tile; splits are cut at multiples of it
constexpr uint32_t kPromptSubRows = 64;    // rows of a work unit of the CUDA-core kernel

struct PromptArgs {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    unsigned char* ws;
    PromptWsLayout l;
    uint64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;  // strides in elements
    uint32_t heads, kv_heads, group, tpt;
    uint32_t q_tokens, kv_tokens;
    uint32_t causal;
    float scale_log2;
    uint32_t vec;  // 16-byte loads of q, k and v rows are aligned
    uint32_t key[5];  // of the plan that the workspace has to hold
    uint32_t* status;
};

// The plan's header, if the plan is one of this geometry; otherwise one without
// items, and PP_DEV_PLAN_MISMATCH from the thread that reports.
__device__ __forceinline__ PromptHeader plan_header(const PromptArgs& a, bool report) {
    PromptHeader h = *reinterpret_cast<const PromptHeader*>(a.ws);
    uint32_t differ = 0;
#pragma unroll
    for (int i = 0; i < 5; ++i) differ |= h.key[i] ^ a.key[i];
    if (differ) {
        h.n_items = h.n_cuts = 0;
        if (report && a.status) atomicOr(a.status, PP_DEV_PLAN_MISMATCH);
    }
    return h;
}

__device__ __forceinline__ uint32_t prompt_visible(const PromptEntry& e, uint32_t token, uint32_t causal) {
    if (!causal) return e.nk;
    const uint64_t v = (uint64_t)e.nk + token + 1;  // keys 0 .. nk - nq + token
    return v > e.nq ? (uint32_t)min((uint64_t)e.nk, v - e.nq) : 0u;
}

// One row by one warp from the keys it sees and nothing else: what a tile does with
// masks does not hold where a masked value is not finite.  bf16 rows on 16-byte
// boundaries.
template <int D>
__device__ __noinline__ void redo_row(const PromptArgs& a, const PromptEntry& e, uint32_t head, uint32_t token,
                                      uint32_t g) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q) + (uint64_t)(e.q0 + token) * a.q_ts +
                        (uint64_t)(head * a.group + g) * a.q_hs;
    const uint32_t end = prompt_visible(e, token, a.causal);
    float m = -__int_as_float(0x7f800000), z = 0.f, acc[E];
#pragma unroll
    for (int c = 0; c < E; ++c) acc[c] = 0.f;
    for (uint32_t n0 = 0; n0 < end; n0 += 32) {
        float s = -__int_as_float(0x7f800000);
        if (n0 + lane < end) {
            const uint16_t* k = reinterpret_cast<const uint16_t*>(a.k) + ((uint64_t)e.k0 + n0 + lane) * a.k_ts +
                                (uint64_t)head * a.k_hs;
            float dot = 0.f;
            for (int c = 0; c < D; c += 2) {
                const uint32_t x = *reinterpret_cast<const uint32_t*>(q + c), y = *reinterpret_cast<const uint32_t*>(k + c);
                dot = fmaf(bf16_lo_to_f32(x), bf16_lo_to_f32(y), dot);
                dot = fmaf(bf16_hi_to_f32(x), bf16_hi_to_f32(y), dot);
            }
            s = dot * a.scale_log2;
        }
        float top = s;
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float mn = fmaxf(m, top), ref = mn == -__int_as_float(0x7f800000) ? 0.f : mn;
        const float f = exp2f(m - ref), p = exp2f(s - ref);
        float sum = p;
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        z = z * f + sum;
        m = mn;
#pragma unroll
        for (int c = 0; c < E; ++c) acc[c] *= f;
        const uint32_t cnt = min(32u, end - n0);
        for (uint32_t i = 0; i < cnt; ++i) {
            const float pi = __shfl_sync(0xffffffffu, p, i);
            const uint16_t* v = reinterpret_cast<const uint16_t*>(a.v) + ((uint64_t)e.k0 + n0 + i) * a.v_ts +
                                (uint64_t)head * a.v_hs;
#pragma unroll
            for (int c = 0; c < E; ++c) acc[c] = fmaf(pi, bf16_lo_to_f32(v[lane + 32 * c]), acc[c]);
        }
    }
    __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out) +
                         ((uint64_t)(e.q0 + token) * a.heads + head * a.group + g) * D;
#pragma unroll
    for (int c = 0; c < E; ++c) out[lane + 32 * c] = __float2bfloat16_rn(acc[c] / z);
}

}  // namespace pp
