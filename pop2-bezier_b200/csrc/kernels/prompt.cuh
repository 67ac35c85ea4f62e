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
    uint32_t kv_tokens;
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

// Whether a row of a tile that is not finite may owe it to keys that it does not see.
// Those in its tile's last key tiles enter P V with P = 0, and 0 * v is not 0 where
// v is NaN or infinite.  A channel is settled, its NaN being the row's own, if one of
// the last keys that the row sees holds a NaN there as well.  By one warp.
template <int D>
__device__ __forceinline__ bool spoiled_by_masked(const PromptArgs& a, const PromptEntry& e, uint32_t head,
                                                  uint32_t token) {
    constexpr int E = D / 32;
    constexpr uint32_t kLook = 32;  // keys it sees that are looked at
    const int lane = threadIdx.x & 31;
    const uint32_t seen = prompt_visible(e, token, a.causal);
    // a later row of the tile is at most tpt - 1 tokens further; key tiles are cut at multiples of their size
    const uint32_t most = min((uint64_t)e.nk, (uint64_t)seen + a.tpt - 1);
    const uint32_t end = min((uint64_t)a.kv_tokens - e.k0, ((uint64_t)most + kPromptKeyTile - 1) / kPromptKeyTile * kPromptKeyTile);
    const uint16_t* v = reinterpret_cast<const uint16_t*>(a.v) + (uint64_t)head * a.v_hs + lane;
    uint32_t open = 0;  // channels lane + 32 c, as bits
#pragma unroll 4
    for (uint32_t n = seen; n < end; ++n)
#pragma unroll
        for (int c = 0; c < E; ++c)
            open |= ((v[((uint64_t)e.k0 + n) * a.v_ts + 32 * c] & 0x7f80u) == 0x7f80u ? 1u : 0u) << c;
    for (uint32_t n = seen; __any_sync(0xffffffffu, open != 0) && n && seen - n < kLook; --n)
#pragma unroll
        for (int c = 0; c < E; ++c)
            if ((v[((uint64_t)e.k0 + n - 1) * a.v_ts + 32 * c] & 0x7fffu) > 0x7f80u) open &= ~(1u << c);
    return __any_sync(0xffffffffu, open != 0);
}

// One row by one warp from the keys it sees and nothing else, if what a tile does
// with masks may have spoiled it.  bf16 rows on 16-byte boundaries.
//
// A row whose own keys hold the NaN stays as it is, and so does one with a NaN in the
// sum of P, which its own scores alone enter: one NaN early in a prompt spoils all
// later rows, and computing them again took a thousand times the call (16384 tokens,
// 16 heads on 4 of 128, 0.9 ms: 880 ms with a token of NaN, now 1.1; 4096 tokens,
// 0.1 ms, with one NaN in v: 76 ms, now 0.7).  What is left is slow, bound by the latency
// of loads that one warp makes: the up to 255 tokens ahead of a lone value that is not
// finite (in the middle of 4096: 11 ms), and rows that see an infinite channel with
// more of it behind their border (all of 4096: 28 ms).
template <int D>
__device__ __noinline__ void redo_row(const PromptArgs& a, const PromptEntry& e, uint32_t head, uint32_t token,
                                      uint32_t g) {
    constexpr int E = D / 32;
    if (!spoiled_by_masked<D>(a, e, head, token)) return;
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
#pragma unroll 8
            for (int c = 0; c < D; c += 8) {
                const uint4 x4 = *reinterpret_cast<const uint4*>(q + c), y4 = *reinterpret_cast<const uint4*>(k + c);
                const uint32_t x[4] = {x4.x, x4.y, x4.z, x4.w}, y[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    dot = fmaf(bf16_lo_to_f32(x[i]), bf16_lo_to_f32(y[i]), dot);
                    dot = fmaf(bf16_hi_to_f32(x[i]), bf16_hi_to_f32(y[i]), dot);
                }
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
#pragma unroll 8
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
