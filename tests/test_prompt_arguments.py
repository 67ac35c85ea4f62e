"""Arguments of the prompt operators that only Python sees: sizes beyond the C ABI's."""
from __future__ import annotations

import pytest
import torch


def test_sizes_beyond_32_bits(pp):
    N = pp._native
    for ok in ((0,), (2**32 - 1, 5), (1, 2, 3)):
        N.check_u32(*ok)
    for bad in ((2**32,), (3, 2**32 + 7), (-1,), (0, -(2**32) + 1)):
        with pytest.raises(pp.PreconditionError):
            N.check_u32(*bad)


@pytest.mark.gpu
def test_sizes_beyond_32_bits_are_refused(pp, cuda):
    """Their lower 32 bits would be small and valid sizes: a head of 2^32 + 100 columns was scored as one of 100."""
    P = pp.PreconditionError
    starts = torch.tensor([0, 10], dtype=torch.int32, device=cuda)
    q = torch.randn(10, 2, 64, device=cuda)
    far = q[:1].expand(2**32 + 10, 2, 64)
    with pytest.raises(P, match="2\\^32"):
        pp.fused_attention.prompt_attention(q, far, far, starts)
    with pytest.raises(P, match="2\\^32"):
        pp.fused_attention.prompt_workspace(q, far, far, 1)
    with pytest.raises(P, match="2\\^32"):
        pp.fused_attention.prompt_workspace(q, q, q, 1, max_ctas=2**32 + 1)
    arena = pp.kv_cache.Int8KvArena.zeros(1, 2, 64, 16, cuda)
    with pytest.raises(P, match="2\\^32"):
        arena.append_prompt(far, far, starts, starts[:1])
    head = torch.empty(1, 2**32 + 100, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(P, match="2\\^32"):
        pp.sampling.token_logprobs(head, torch.zeros(1, dtype=torch.int32, device=cuda))
    rows = q[:1, 0].expand(2**32 + 1, 64)
    with pytest.raises(P, match="2\\^32"):
        pp.sampling.token_logprobs(rows, torch.zeros(1, dtype=torch.int32, device=cuda))
