// C ABI of the prompt path: attention over packed sequences, the append of
// packed prompts and the log probabilities of given tokens.  Checks first;
// nothing is launched when one fails.
#include <cmath>
#include <cstdint>
#include <cstring>

#include "internal.h"

namespace {

using pp::fail_fmt;

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// Geometry of a prompt; `tensors` also checks q, k and v.
int32_t check_prompt(const PpPrompt* p, bool tensors, const char* what) {
    if (!p || p->struct_size < sizeof(PpPrompt)) return fail_fmt(PP_STATUS_PRECONDITION, "%s: PpPrompt missing", what);
    if (p->sequences == 0 || p->heads == 0 || p->kv_heads == 0 || p->heads % p->kv_heads != 0 ||
        p->heads / p->kv_heads > 64 || (p->head_dim != 64 && p->head_dim != 128) ||
        (p->dtype != PP_DTYPE_F32 && p->dtype != PP_DTYPE_BF16))
        return fail_fmt(PP_STATUS_PRECONDITION,
                        "prompt attention requires F32/BF16 [tokens,heads,64|128] with heads a multiple (1..64) of the K/V "
                        "heads: sequences=%u heads=%u kv_heads=%u head_dim=%u dtype=%d",
                        p->sequences, p->heads, p->kv_heads, p->head_dim, p->dtype);
    const uint32_t entry_tokens = 2 * (128 / (p->heads / p->kv_heads));
    if (p->q_tokens > 0x7fffff00u || p->kv_tokens > 0x7fffff00u || p->sequences > 0x7fffff00u || p->max_ctas > 65536u ||
        p->heads > 65535u ||
        ((uint64_t)p->q_tokens / entry_tokens + p->sequences + 2 * 65536ull) * p->kv_heads > 0x3fffffffull)
        return fail_fmt(PP_STATUS_PRECONDITION, "prompt attention dimensions overflow: q_tokens=%u kv_tokens=%u sequences=%u",
                        p->q_tokens, p->kv_tokens, p->sequences);
    if (!(p->softmax_scale >= 0.f) || !std::isfinite(p->softmax_scale))
        return fail_fmt(PP_STATUS_PRECONDITION, "softmax_scale must be finite and >= 0");
    if (!tensors) return PP_STATUS_OK;
    if ((p->q_tokens && !p->q) || (p->kv_tokens && (!p->k || !p->v)))
        return fail_fmt(PP_STATUS_PRECONDITION, "%s: NULL q, k or v", what);
    const uintptr_t elem = p->dtype == PP_DTYPE_F32 ? 4 : 2;
    if (!aligned(p->q, elem) || !aligned(p->k, elem) || !aligned(p->v, elem))
        return fail_fmt(PP_STATUS_PRECONDITION, "%s: misaligned q, k or v", what);
    const uint64_t strides[6] = {p->q_token_stride, p->q_head_stride, p->k_token_stride,
                                 p->k_head_stride,  p->v_token_stride, p->v_head_stride};
    for (uint64_t s : strides)
        if (s >= (1ull << 36)) return fail_fmt(PP_STATUS_PRECONDITION, "%s: strides overflow", what);
    return PP_STATUS_OK;
}

int32_t prompt_ctas(const PpPrompt& p, uint32_t* ctas, uint32_t* sms) {
    int32_t s = pp::device_sms(sms);
    *ctas = p.max_ctas ? p.max_ctas : *sms;
    return s;
}

int32_t prepare_prompt(const PpPrompt* prompt, const uint32_t* q_starts, const uint32_t* kv_starts, void* workspace,
                       size_t ws_bytes, uint32_t* status, bool tensors, pp::PromptLaunch& L, const char* what) {
    int32_t s;
    if ((s = check_prompt(prompt, tensors, what))) return s;
    if (!q_starts) return fail_fmt(PP_STATUS_PRECONDITION, "%s: q_starts is NULL", what);
    if (!aligned(q_starts, 4) || !aligned(kv_starts, 4) || !aligned(status, 4))
        return fail_fmt(PP_STATUS_PRECONDITION, "%s: starts and status must be 4-byte aligned", what);
    uint32_t ctas = 0;
    L = pp::PromptLaunch{};
    L.g = *prompt;
    if ((s = prompt_ctas(L.g, &ctas, &L.num_sms))) return s;
    L.layout = pp::prompt_ws_layout(L.g.sequences, L.g.q_tokens, L.g.heads, L.g.kv_heads, L.g.head_dim, ctas);
    if (!workspace) return fail_fmt(PP_STATUS_PRECONDITION, "%s: workspace is NULL", what);
    if (!aligned(workspace, 256)) return fail_fmt(PP_STATUS_PRECONDITION, "%s: workspace must be 256-byte aligned", what);
    if (ws_bytes < L.layout.total)
        return fail_fmt(PP_STATUS_PRECONDITION, "%s: workspace too small (%zu < %zu bytes)", what, ws_bytes, L.layout.total);
    L.q_starts = q_starts;
    L.kv_starts = kv_starts ? kv_starts : q_starts;
    L.ws = static_cast<unsigned char*>(workspace);
    L.status = status;
    const float scale = L.g.softmax_scale > 0.f ? L.g.softmax_scale
                                                : (L.g.head_dim == 64 ? 0.125f : (float)(1.0 / std::sqrt(128.0)));
    L.scale_log2 = scale * 1.4426950408889634f;
    return PP_STATUS_OK;
}

}  // namespace

extern "C" {

size_t pp_b200_prompt_workspace_size(const PpPrompt* prompt) {
    if (check_prompt(prompt, false, "prompt_workspace_size") != PP_STATUS_OK) return 0;
    uint32_t ctas = 0, sms = 0;
    if (prompt_ctas(*prompt, &ctas, &sms) != PP_STATUS_OK) ctas = prompt->max_ctas ? prompt->max_ctas : 1024;
    return pp::prompt_ws_layout(prompt->sequences, prompt->q_tokens, prompt->heads, prompt->kv_heads, prompt->head_dim,
                                ctas).total;
}

int32_t pp_b200_plan_prompt(const PpPrompt* prompt, const uint32_t* q_starts, const uint32_t* kv_starts,
                            void* workspace, size_t workspace_bytes, uint32_t* status, void* stream) {
    pp::PromptLaunch L;
    int32_t s = prepare_prompt(prompt, q_starts, kv_starts, workspace, workspace_bytes, status, false, L, "plan_prompt");
    if (s) return s;
    return pp::cuda_status(pp::launch_prompt_plan(L, (cudaStream_t)stream), "prompt plan launch");
}

int32_t pp_b200_prompt_attention(const PpPrompt* prompt, const uint32_t* q_starts, const uint32_t* kv_starts,
                                 void* out, void* workspace, size_t workspace_bytes, uint32_t* status, void* stream) {
    pp::PromptLaunch L;
    int32_t s = prepare_prompt(prompt, q_starts, kv_starts, workspace, workspace_bytes, status, true, L,
                               "prompt_attention");
    if (s) return s;
    if (L.g.flags & ~PP_ATTN_PLAN_READY) return fail_fmt(PP_STATUS_PRECONDITION, "prompt_attention: unknown flags 0x%x", L.g.flags);
    if (L.g.q_tokens == 0)  // no rows, but starts that the plan checks
        return L.g.flags & PP_ATTN_PLAN_READY
                   ? PP_STATUS_OK
                   : pp::cuda_status(pp::launch_prompt_plan(L, (cudaStream_t)stream), "prompt plan launch");
    if (!out || !aligned(out, 16)) return fail_fmt(PP_STATUS_PRECONDITION, "prompt_attention: out must be 16-byte aligned");
    L.out = out;
    const uint64_t elem = L.g.dtype == PP_DTYPE_F32 ? 4 : 2;
    // a dimension of one element has no stride worth checking
    if (L.g.q_tokens == 1) L.g.q_token_stride = (uint64_t)L.g.heads * L.g.head_dim;
    if (L.g.heads == 1) L.g.q_head_stride = L.g.head_dim;
    if (L.g.kv_tokens <= 1) L.g.k_token_stride = L.g.v_token_stride = (uint64_t)L.g.kv_heads * L.g.head_dim;
    if (L.g.kv_heads == 1) L.g.k_head_stride = L.g.v_head_stride = L.g.head_dim;
    L.vec = aligned(L.g.q, 16) && aligned(L.g.k, 16) && aligned(L.g.v, 16) &&
            (L.g.q_token_stride * elem) % 16 == 0 && (L.g.q_head_stride * elem) % 16 == 0 &&
            (L.g.k_token_stride * elem) % 16 == 0 && (L.g.k_head_stride * elem) % 16 == 0 &&
            (L.g.v_token_stride * elem) % 16 == 0 && (L.g.v_head_stride * elem) % 16 == 0;
    cudaStream_t st = (cudaStream_t)stream;
    // The tensor cores take bf16 rows on 16-byte boundaries (what the tensor
    // copies need; a stride of 0, as `expand` makes, is none they take).
    const bool tc = L.g.dtype == PP_DTYPE_BF16 && L.vec && L.g.kv_tokens && L.g.q_token_stride && L.g.q_head_stride &&
                    L.g.k_token_stride && L.g.k_head_stride && L.g.v_token_stride && L.g.v_head_stride;
    CUtensorMap map_q{}, map_k{}, map_v{};
    if (tc) {
        const uint32_t d = L.g.head_dim, group = L.g.heads / L.g.kv_heads;
        const uint64_t q_dims[4] = {d, group, L.g.q_tokens, L.g.kv_heads};
        const uint64_t q_st[3] = {L.g.q_head_stride * 2, L.g.q_token_stride * 2, L.g.q_head_stride * 2 * group};
        const uint32_t q_box[4] = {64, group, 128 / group, 1}, kv_box[3] = {64, 128, 1};
        const uint64_t kv_dims[3] = {d, L.g.kv_tokens, L.g.kv_heads};
        const uint64_t k_st[2] = {L.g.k_token_stride * 2, L.g.k_head_stride * 2};
        const uint64_t v_st[2] = {L.g.v_token_stride * 2, L.g.v_head_stride * 2};
        const CUtensorMapDataType bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        if ((s = pp::encode_tiled(&map_q, bf, 4, L.g.q, q_dims, q_st, q_box, "prompt q")) ||
            (s = pp::encode_tiled(&map_k, bf, 3, L.g.k, kv_dims, k_st, kv_box, "prompt k")) ||
            (s = pp::encode_tiled(&map_v, bf, 3, L.g.v, kv_dims, v_st, kv_box, "prompt v")))
            return s;
    }
    if (!(L.g.flags & PP_ATTN_PLAN_READY) && (s = pp::cuda_status(pp::launch_prompt_plan(L, st), "prompt plan launch")))
        return s;
    s = pp::cuda_status(tc ? pp::launch_prompt_tc(L, map_q, map_k, map_v, st) : pp::launch_prompt_rows(L, st),
                        "prompt attention launch");
    // no entry of so few keys is cut (prompt.cu)
    if (s || L.g.kv_tokens <= pp::prompt_uncut_keys()) return s;
    return pp::cuda_status(pp::launch_prompt_merge(L, st), "prompt merge launch");
}

int32_t pp_b200_prompt_append(const PpKvArena* arena, const void* k, const void* v, int32_t dtype, uint32_t tokens,
                              uint64_t k_token_stride, uint64_t k_head_stride, uint64_t v_token_stride,
                              uint64_t v_head_stride, const uint32_t* starts, const uint32_t* offsets,
                              uint32_t* status, void* stream) {
    int32_t s;
    if ((s = pp::check_arena(arena, "prompt_append"))) return s;
    if (dtype != PP_DTYPE_F32 && dtype != PP_DTYPE_BF16)
        return fail_fmt(PP_STATUS_PRECONDITION, "prompt_append: unsupported dtype %d", dtype);
    if (tokens > 0x7fffff00u || (k_token_stride | k_head_stride | v_token_stride | v_head_stride) >= (1ull << 36))
        return fail_fmt(PP_STATUS_PRECONDITION, "prompt_append: dimensions overflow: tokens=%u", tokens);
    if (!starts || !offsets || !aligned(starts, 4) || !aligned(offsets, 4) || !aligned(status, 4))
        return fail_fmt(PP_STATUS_PRECONDITION, "prompt_append: starts, offsets and status must be 4-byte aligned");
    pp::PromptAppendLaunch P{};
    if ((s = pp::device_sms(&P.num_sms))) return s;
    if (tokens == 0 && !status) return PP_STATUS_OK;  // nothing to append, and nowhere to report bad starts
    const uint64_t elem = dtype == PP_DTYPE_F32 ? 4 : 2;
    if ((tokens && (!k || !v)) || !aligned(k, elem) || !aligned(v, elem))
        return fail_fmt(PP_STATUS_PRECONDITION, "prompt_append: NULL or misaligned K/V");
    P.arena = arena;
    P.k = k;
    P.v = v;
    P.bf16 = dtype == PP_DTYPE_BF16;
    P.tokens = tokens;
    P.k_ts = k_token_stride;
    P.k_hs = k_head_stride;
    P.v_ts = v_token_stride;
    P.v_hs = v_head_stride;
    P.starts = starts;
    P.offsets = offsets;
    P.status = status;
    P.vec = aligned(k, 16) && aligned(v, 16) && (k_token_stride * elem) % 16 == 0 && (k_head_stride * elem) % 16 == 0 &&
            (v_token_stride * elem) % 16 == 0 && (v_head_stride * elem) % 16 == 0;
    return pp::cuda_status(pp::launch_prompt_append(P, (cudaStream_t)stream), "prompt append launch");
}

int32_t pp_b200_token_logprobs(const void* logits, int32_t dtype, uint32_t rows, uint32_t choices,
                               uint64_t row_stride, const int32_t* targets, const uint32_t* bounds, uint32_t top,
                               float* logprob, float* entropy, uint32_t* rank, uint32_t* top_ids,
                               float* top_logprobs, uint32_t* status, void* stream) {
    if (dtype != PP_DTYPE_F32 && dtype != PP_DTYPE_BF16)
        return fail_fmt(PP_STATUS_PRECONDITION, "token logprobs: unsupported dtype %d", dtype);
    if (choices == 0 || choices > 0x7fffff00u || rows > 0x7fffffffu || top > 32)
        return fail_fmt(PP_STATUS_PRECONDITION,
                        "token logprobs need a nonempty head and at most 32 alternatives: rows=%u choices=%u top=%u", rows,
                        choices, top);
    if (row_stride >= (1ull << 36))
        return fail_fmt(PP_STATUS_PRECONDITION, "token logprobs: row stride %llu overflows", (unsigned long long)row_stride);
    pp::LogprobsLaunch L{};
    int32_t s;
    if ((s = pp::device_sms(&L.num_sms))) return s;
    if (rows == 0) return PP_STATUS_OK;
    if (!logits || !targets || !logprob || !entropy || !rank || (top && (!top_ids || !top_logprobs)))
        return fail_fmt(PP_STATUS_PRECONDITION, "token logprobs: NULL pointer");
    if (!aligned(logits, dtype == PP_DTYPE_F32 ? 4 : 2) || !aligned(targets, 4) || !aligned(bounds, 4) ||
        !aligned(logprob, 4) || !aligned(entropy, 4) || !aligned(rank, 4) || !aligned(top_ids, 4) ||
        !aligned(top_logprobs, 4) || !aligned(status, 4))
        return fail_fmt(PP_STATUS_PRECONDITION, "token logprobs: misaligned pointer");
    L.logits = logits;
    L.bf16 = dtype == PP_DTYPE_BF16;
    L.rows = rows;
    L.choices = choices;
    L.top = top;
    L.row_stride = row_stride;
    L.targets = targets;
    L.bounds = bounds;
    L.logprob = logprob;
    L.entropy = entropy;
    L.rank = rank;
    L.top_ids = top_ids;
    L.top_logprobs = top_logprobs;
    L.status = status;
    return pp::cuda_status(pp::launch_token_logprobs(L, (cudaStream_t)stream), "token logprobs launch");
}

}  // extern "C"
