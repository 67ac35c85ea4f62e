"""Float-KV fused decode attention over the C ABI (device tensors only).

Mirrors fused_attention::decode_attention (app/src/model/fused_attention.rs:
8-33): q [rows, 1, d] (or [rows, d]), K/V [rows, length, d] in bf16 or f32
with dense channel and token strides (any row stride), optional per-branch
lengths, `heads` heads per branch and the reference's split_tokens.  Returns
f32 [rows, 1, d] like the reference.  The reference's errors are raised as
PreconditionError with its messages; there is no CPU branch (the reference
bails with "select ordinary attention for CPU").

Differences, all documented at the call:
  * head_dim 128 is accepted besides 64, and bf16 q besides f32;
  * the key length is not capped at 1024;
  * split_tokens == 0 selects the balanced stream-K plan instead of one CTA
    per row; a non-zero split_tokens is clamped to [32, 1024] as the
    reference does.  Results agree within f32 reassociation for any split.

prompt_attention is the prefill side: every token of a batch of packed prompts
attends to its own sequence (the reference's ordinary causal attention,
app/src/model/mod.rs:716-720, with K/V shared by groups of query heads).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _native as N
from . import int8_kv_ops as ops

_MSG_SHAPE = "fused decode attention requires F32[batch*heads,1,64] and same-device BF16/F32 K/V"
_MSG_STRIDE = "fused attention requires dense width and token strides"
_MSG_LENGTHS = "fused attention row lengths require same-device U32[batch]"


def kv_struct(k: torch.Tensor, v: torch.Tensor, heads: int) -> N.PpFloatKv:
    rows, n, d = k.shape
    g = N.PpFloatKv()
    g.struct_size = C.sizeof(N.PpFloatKv)
    g.rows, g.heads, g.head_dim, g.tokens = rows, heads, d, n
    g.dtype = N.DTYPE_F32 if k.dtype == torch.float32 else N.DTYPE_BF16
    g.k_row_stride, g.v_row_stride = k.stride(0), v.stride(0)
    g.k, g.v = k.data_ptr(), v.data_ptr()
    return g


def _check(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor | None, heads: int) -> None:
    """The checks of fused_attention.rs:10-25 (head_dim 64 or 128)."""
    for t in (q, k, v, lengths):
        if t is not None and not t.is_cuda:
            raise N.PreconditionError("NVIDIA fused attention needs CUDA; use ordinary attention on this backend")
    if q.dim() == 2:
        q = q.unsqueeze(1)
    if q.dim() != 3 or k.dim() != 3:
        raise N.PreconditionError(_MSG_SHAPE)
    rows, query, width = q.shape
    key_rows, length, key_width = k.shape
    if heads <= 0 or rows == 0 or rows % heads != 0 or query != 1 or width not in (64, 128) or key_rows != rows \
            or key_width != width or length == 0 or tuple(v.shape) != tuple(k.shape) \
            or q.dtype not in (torch.float32, torch.bfloat16) or k.dtype not in (torch.float32, torch.bfloat16) \
            or k.dtype != v.dtype or q.device != k.device or q.device != v.device:
        raise N.PreconditionError(_MSG_SHAPE)
    for t in (k, v):
        if t.stride(2) != 1 or t.stride(1) != width:
            raise N.PreconditionError(_MSG_STRIDE)
    if q.stride(2) != 1:
        raise N.PreconditionError(_MSG_STRIDE)
    if lengths is not None:
        if lengths.dim() != 1 or lengths.numel() != rows // heads or lengths.dtype not in (torch.int32, torch.uint32) \
                or not lengths.is_contiguous() or lengths.device != q.device:
            raise N.PreconditionError(_MSG_LENGTHS)


def workspace_bytes(kv: N.PpFloatKv, params: N.PpAttnParams) -> int:
    return int(N.lib.pp_b200_float_attention_workspace_size(C.byref(kv), C.byref(params)))


def plan_ragged(k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor | None, heads: int, workspace: torch.Tensor,
                *, split_tokens: int = 0, q_dtype: torch.dtype = torch.float32) -> None:
    """Writes the split plan for these lengths into `workspace` (reused by
    calls with plan_ready=True, e.g. by every layer of one decode step)."""
    kv = kv_struct(k, v, heads)
    params = ops.attn_params(split_tokens=split_tokens, q_dtype=q_dtype)
    N.check(N.lib.pp_b200_plan_ragged_float(C.byref(kv), C.byref(params), ops._ptr(lengths), ops._ptr(workspace),
                                            workspace.numel(), ops._stream(k)))


def decode_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor | None, heads: int,
                     split_tokens: int = 0, *, out_dtype: torch.dtype = torch.float32, softmax_scale: float = 0.0,
                     workspace: torch.Tensor | None = None, plan_ready: bool = False,
                     prefetch_history: bool = False, status: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Fused float-KV decode attention; returns [rows, 1, d] (out_dtype, f32
    by default as the reference)."""
    _check(q, k, v, lengths, heads)
    rows, d = k.shape[0], k.shape[2]
    q_stride = q.stride(0)
    kv = kv_struct(k, v, heads)
    params = ops.attn_params(split_tokens=split_tokens, q_dtype=q.dtype, out_dtype=out_dtype,
                             softmax_scale=softmax_scale, plan_ready=plan_ready, prefetch_history=prefetch_history)
    if workspace is None:
        workspace = torch.empty(workspace_bytes(kv, params), dtype=torch.uint8, device=q.device)
    if out is None:
        out = torch.empty((rows, 1, d), dtype=out_dtype, device=q.device)
    N.check(N.lib.pp_b200_decode_attention_float(C.byref(kv), C.byref(params), ops._ptr(q), q_stride,
                                                 ops._ptr(lengths), ops._ptr(out), ops._ptr(workspace),
                                                 workspace.numel(), ops._ptr(status), ops._stream(q)))
    return out


def prepare_optional_kernels(device: torch.device | int, fusion: bool, split_k: bool, *,
                             dtype: torch.dtype = torch.bfloat16, head_width: int = 64, ffn_hidden: int = 0) -> None:
    """PrimitiveModel::prepare_optional_kernels (mod.rs:440-460): on-device
    zero-input checks of the fused attention (and SwiGLU with `fusion`);
    raises PreconditionError with the reference's messages."""
    idx = device.index if isinstance(device, torch.device) else int(device)
    code = N.DTYPE_F32 if dtype == torch.float32 else N.DTYPE_BF16
    N.check(N.lib.pp_b200_prepare_optional(0 if idx is None else idx, int(fusion), int(split_k), code, head_width,
                                           ffn_hidden))


_MSG_PROMPT = ("prompt attention requires CUDA BF16/F32 q [tokens,heads,64|128] and k, v [tokens,kv_heads,64|128] of one "
               "type and device, heads a multiple (1..64) of kv_heads, head_dim contiguous")
_MSG_STARTS = "prompt starts must be contiguous same-device U32 [sequences + 1]"


def _starts(t: torch.Tensor, n: int | None, device: torch.device) -> int:
    if t.dim() != 1 or t.numel() < 2 or (n is not None and t.numel() != n + 1) \
            or t.dtype not in (torch.int32, torch.uint32) or not t.is_contiguous() or t.device != device:
        raise N.PreconditionError(_MSG_STARTS)
    return t.numel() - 1


_PROMPT_DTYPES = {torch.float32: N.DTYPE_F32, torch.bfloat16: N.DTYPE_BF16}


def prompt_struct(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, sequences: int, *, causal: bool = True,
                  softmax_scale: float = 0.0, plan_ready: bool = False, max_ctas: int = 0) -> N.PpPrompt:
    """The C ABI's geometry of packed prompts, after its checks."""
    kshape, dt = k.shape, q.dtype
    if q.dim() != 3 or len(kshape) != 3 or v.shape != kshape:
        raise N.PreconditionError(_MSG_PROMPT)
    tokens, heads, d = q.shape
    kv_tokens, kv_heads, kd = kshape
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    code = _PROMPT_DTYPES.get(dt)
    dev = q.get_device() if q.is_cuda else -1
    if dev < 0 or k.get_device() != dev or v.get_device() != dev or kd != d or (d != 64 and d != 128) or code is None \
            or k.dtype != dt or v.dtype != dt or heads == 0 or kv_heads == 0 or heads % kv_heads or heads > 64 * kv_heads \
            or qs[2] != 1 or ks[2] != 1 or vs[2] != 1:
        raise N.PreconditionError(_MSG_PROMPT)
    N.check_u32(sequences, tokens, kv_tokens, max_ctas)
    return N.PpPrompt(_PROMPT_BYTES, sequences, heads, kv_heads, d, code, tokens, kv_tokens, 1 if causal else 0,
                      softmax_scale, N.ATTN_PLAN_READY if plan_ready else 0, max_ctas, qs[0], qs[1], ks[0], ks[1], vs[0],
                      vs[1], q.data_ptr(), k.data_ptr(), v.data_ptr())


_PROMPT_BYTES = C.sizeof(N.PpPrompt)


def prompt_workspace(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, sequences: int, *, max_ctas: int = 0
                     ) -> torch.Tensor:
    """A workspace for plan_prompt / prompt_attention over tensors of these
    shapes and that many sequences.  Calls that may run at the same time need
    one each."""
    g = prompt_struct(q, k, v, sequences, max_ctas=max_ctas)
    with ops._here(q):
        return torch.empty(int(N.lib.pp_b200_prompt_workspace_size(C.byref(g))), dtype=torch.uint8, device=q.device)


def plan_prompt(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_starts: torch.Tensor, workspace: torch.Tensor, *,
                kv_starts: torch.Tensor | None = None, causal: bool = True, max_ctas: int = 0,
                status: torch.Tensor | None = None) -> None:
    """Writes the work list of these sequences into `workspace`, for the
    prompt_attention calls with plan_ready=True that follow: every layer of a
    prefill has the same shapes and lengths.  A call of another shape,
    causality, max_ctas or number of sequences writes nothing and sets
    DEV_PLAN_MISMATCH in its status word."""
    n = _starts(q_starts, None, q.device)
    if kv_starts is not None:
        _starts(kv_starts, n, q.device)
    g = prompt_struct(q, k, v, n, causal=causal, max_ctas=max_ctas)
    _prompt_buffers(q, workspace, status)
    with ops._here(q):
        N.check(N.lib.pp_b200_plan_prompt(C.byref(g), q_starts.data_ptr(), ops._ptr(kv_starts), workspace.data_ptr(),
                                          workspace.numel(), ops._ptr(status), ops._stream(q)))


def _prompt_buffers(q: torch.Tensor, workspace: torch.Tensor | None, status: torch.Tensor | None) -> None:
    if workspace is not None and (workspace.dtype != torch.uint8 or not workspace.is_contiguous()
                                  or workspace.device != q.device):
        raise N.PreconditionError("prompt workspace must be a contiguous same-device byte tensor")
    ops.check_status(status, q.device)


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_starts: torch.Tensor, *,
                     kv_starts: torch.Tensor | None = None, causal: bool = True, softmax_scale: float = 0.0,
                     workspace: torch.Tensor | None = None, plan_ready: bool = False, max_ctas: int = 0,
                     status: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of packed prompts; returns [tokens, heads, head_dim] of q's type.

    q [tokens, heads, d], k and v [kv_tokens, kv_heads, d], bf16 or f32, any
    token and head strides (bf16 on 16-byte boundaries and without strides of 0
    runs on the tensor cores, everything else on the CUDA cores, which takes
    about ten times as long: pass shared K/V heads as kv_heads, not by expand);
    q_starts int32/uint32 [sequences + 1] on the
    device: sequence s holds the query tokens q_starts[s] .. q_starts[s + 1].
    kv_starts does the same for the keys (default: the same tokens).  A causal
    query i of n, with m keys, sees keys 0 .. m - n + i: with more keys than
    queries it continues a sequence whose first m - n tokens came before (a
    later chunk of a prompt, or a single token).  A query that sees no key
    gives NaN; rows of `out` that no sequence holds are left as they were, and
    `out` shares no memory with q, k and v.
    softmax_scale 0: 0.125 at d = 64, 1/sqrt(d) otherwise.  A status word gets
    DEV_LENGTH_RANGE when the starts decrease or pass the tensors' ends, and
    DEV_PLAN_MISMATCH when plan_ready finds no plan of this geometry in the
    workspace (in both cases nothing is written)."""
    n = _starts(q_starts, None, q.device)
    if kv_starts is not None:
        _starts(kv_starts, n, q.device)
    g = prompt_struct(q, k, v, n, causal=causal, softmax_scale=softmax_scale, plan_ready=plan_ready, max_ctas=max_ctas)
    _prompt_buffers(q, workspace, status)
    if plan_ready and workspace is None:
        raise N.PreconditionError("plan_ready needs the workspace that plan_prompt wrote")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous():
        raise N.PreconditionError("prompt attention writes a dense [tokens,heads,head_dim] of q's type and device")
    with ops._here(q):
        if workspace is None:
            workspace = torch.empty(N.lib.pp_b200_prompt_workspace_size(C.byref(g)), dtype=torch.uint8, device=q.device)
        N.check(N.lib.pp_b200_prompt_attention(C.byref(g), q_starts.data_ptr(), ops._ptr(kv_starts), out.data_ptr(),
                                               workspace.data_ptr(), workspace.numel(), ops._ptr(status),
                                               ops._stream(q)))
    return out
