/*
 * pp_b200_prompt.h -- geometry of a batch of packed prompts, for the prompt
 * entry points of pp_b200.h (which includes this file).
 */
#ifndef PP_B200_PROMPT_H
#define PP_B200_PROMPT_H

#include <stdint.h>

/* A batch of packed sequences for pp_b200_prompt_attention.  The query tokens
 * of all sequences lie one after another, and so do their keys and values:
 *   q     [q_tokens, heads, head_dim]
 *   k, v  [kv_tokens, kv_heads, head_dim]
 * of `dtype`, head_dim contiguous, with any token and head strides (in
 * elements), so that a view of a QKV projection or of [heads, tokens,
 * head_dim] planes is passed as is (bf16 on 16-byte boundaries and without
 * strides of 0 runs on the tensor cores, everything else on the CUDA cores).
 * Query head h reads K/V head h / (heads / kv_heads).  q_tokens and kv_tokens
 * are the rows that the tensors hold; the sequences' own lengths are device
 * data. */
typedef struct PpPrompt {
    uint32_t struct_size; /* sizeof(PpPrompt) */
    uint32_t sequences;
    uint32_t heads;    /* query heads */
    uint32_t kv_heads; /* divides heads; at most 64 query heads share one */
    uint32_t head_dim; /* 64 or 128 */
    int32_t dtype;     /* PP_DTYPE_F32 or PP_DTYPE_BF16: q, k, v and out */
    uint32_t q_tokens;
    uint32_t kv_tokens;
    uint32_t causal;     /* 0: a token sees all keys of its sequence */
    float softmax_scale; /* 0: 0.125 at head_dim 64, f32(1/sqrt(d)) otherwise */
    uint32_t flags;      /* PP_ATTN_PLAN_READY */
    uint32_t max_ctas;   /* 0: one CTA per SM */
    uint64_t q_token_stride, q_head_stride;
    uint64_t k_token_stride, k_head_stride;
    uint64_t v_token_stride, v_head_stride;
    const void* q;
    const void* k;
    const void* v;
} PpPrompt;

#endif /* PP_B200_PROMPT_H */
