"""Device sampling and scoring after the output heads, on the C ABI.

renyi_sample mirrors fused_sampling::sample (app/src/inference/
fused_sampling.rs:69-90): Rényi-entropy truncated sampling with classifier-
free guidance, one logical row per block, bit-identical to the reference's
pp_renyi_sample.

token_logprobs scores given tokens under the same heads: log probability,
rank, entropy of the row and its best alternatives, as teacher-forced
comparisons of two models read them (app/src/bin/kv_int8_acceptance.rs:60-219).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as N
from . import int8_kv_ops as ops


def renyi_sample(raw: torch.Tensor, uniforms: torch.Tensor, bounds: torch.Tensor, alpha: float, cfg: float,
                 guidance: int, offset: int, *, out: torch.Tensor | None = None):
    """raw f32 [batch*guidance, choices]; uniforms f32 [batch, 1]; bounds u32
    (or i32) [batch, 2] = (start, count).  Returns (tokens, ok, support), each
    [batch, 1] u32 views of one [3, batch] buffer, like the reference."""
    ops._require_cuda(raw, uniforms, bounds)
    if raw.dim() != 2 or guidance not in (1, 2) or raw.shape[0] == 0 or raw.shape[0] % guidance \
            or not 1 <= raw.shape[1] <= 2048:
        raise N.PreconditionError(
            "fused sampler needs 1/2 guidance rows and a nonempty head of at most 2048 choices")
    batch = raw.shape[0] // guidance
    if uniforms.numel() != batch or bounds.numel() != 2 * batch:
        raise N.PreconditionError("fused sampler logical row, uniform or bounds shape mismatch")
    if raw.dtype != torch.float32 or uniforms.dtype != torch.float32 or bounds.dtype not in (torch.int32,
                                                                                             torch.uint32):
        raise N.PreconditionError("fused sampler expects FP32 logits/uniforms and U32 bounds")
    for t in (raw, uniforms, bounds):
        if not t.is_contiguous():
            raise N.PreconditionError("fused sampler inputs must be contiguous; nonzero view offsets are supported")
    if out is None:
        out = torch.empty((3, batch), dtype=torch.int32, device=raw.device)
    N.check(N.lib.pp_b200_renyi_sample(ops._ptr(raw), ops._ptr(uniforms), ops._ptr(bounds), ops._ptr(out), batch,
                                       raw.shape[1], guidance, float(alpha), float(cfg), int(offset),
                                       ops._stream(raw)))
    return out[0].view(batch, 1), out[1].view(batch, 1), out[2].view(batch, 1)


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor  # f32 [rows]
    entropy: torch.Tensor  # f32 [rows], nats
    rank: torch.Tensor  # int32 [rows], 0 for the best
    top_ids: torch.Tensor | None  # int32 [rows, top], -1 where there is none
    top_logprobs: torch.Tensor | None  # f32 [rows, top]


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, *, top: int = 0, bounds: torch.Tensor | None = None,
                   status: torch.Tensor | None = None) -> TokenLogprobs:
    """Scores targets (int32 [rows], columns of their rows; -1: none) under
    logits f32/bf16 [rows, choices] (any row stride): log probability, rank,
    entropy and the `top` (at most 32) best alternatives.

    bounds, u32 (or i32) [rows, 2] = (start, count) as renyi_sample's, limits
    each row to a window of legal columns.  A target outside it has log
    probability -inf and the window's size as its rank.  Alternatives are
    ordered by (logit descending, column ascending); columns whose logit is
    -inf are none.  An empty window gives NaN and no alternatives, and so does
    one outside the choices, which also sets DEV_WINDOW_RANGE in the status
    word.  NaN or +inf in the window makes log probabilities and entropy NaN.
    """
    ops._require_cuda(logits, targets, bounds, status)
    if logits.dim() != 2 or logits.shape[1] == 0 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise N.PreconditionError("token logprobs need logits [rows, choices] with contiguous rows and a nonempty head")
    rows, choices = logits.shape
    N.check_u32(rows, choices)
    if targets.dim() != 1 or targets.numel() != rows or targets.dtype != torch.int32 or not targets.is_contiguous():
        raise N.PreconditionError("token logprobs need one contiguous I32 target a row")
    if bounds is not None and (bounds.numel() != 2 * rows or bounds.dtype not in (torch.int32, torch.uint32)
                               or not bounds.is_contiguous()):
        raise N.PreconditionError("token logprobs bounds must be contiguous U32 [rows, 2]")
    if not 0 <= top <= 32:
        raise N.PreconditionError("token logprobs give at most 32 alternatives")
    ops.check_status(status, logits.device)
    code = ops._dtype_code(logits, "logits")
    stride = logits.stride(0) if rows > 1 else choices
    dev = logits.device
    logprob = torch.empty(rows, dtype=torch.float32, device=dev)
    entropy, rank = torch.empty_like(logprob), torch.empty_like(targets)
    ids = torch.empty((rows, top), dtype=torch.int32, device=dev) if top else None
    best = torch.empty((rows, top), dtype=torch.float32, device=dev) if top else None
    with ops._here(logits):
        N.check(N.lib.pp_b200_token_logprobs(
            logits.data_ptr(), code, rows, choices, stride, targets.data_ptr(), ops._ptr(bounds), top,
            logprob.data_ptr(), entropy.data_ptr(), rank.data_ptr(), ops._ptr(ids), ops._ptr(best),
            ops._ptr(status), ops._stream(logits)))
    return TokenLogprobs(logprob, entropy, rank, ids, best)
