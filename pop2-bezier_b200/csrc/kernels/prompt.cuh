// Shared by the prompt attention kernels: the work list in the workspace and
// the merge of a row that was cut along its keys.
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
    uint32_t* status;
};

__device__ __forceinline__ uint32_t prompt_visible(const PromptEntry& e, uint32_t token, uint32_t causal) {
    if (!causal) return e.nk;
    const uint64_t v = (uint64_t)e.nk + token + 1;  // keys 0 .. nk - nq + token
    return v > e.nq ? (uint32_t)min((uint64_t)e.nk, v - e.nq) : 0u;
}

__device__ __forceinline__ uint32_t ld_acquire(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

}  // namespace pp
