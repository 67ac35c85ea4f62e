"""Arguments of the prompt operators at their ends: sizes beyond 32 bits, and none."""
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


@pytest.mark.gpu
@pytest.mark.parametrize("starts", [[0, 5, 5], [0, 0, 1], [3, 2, 0]])
def test_starts_are_checked_without_tokens(pp, cuda, starts):
    """Empty tensors hold no token that starts may name."""
    N = pp._native
    bad, none = (torch.tensor(s, dtype=torch.int32, device=cuda) for s in (starts, [0, 0, 0]))
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    empty, keys = torch.empty(0, 2, 64, device=cuda), torch.randn(7, 2, 64, device=cuda)
    fa = pp.fused_attention
    ws = fa.prompt_workspace(empty, keys, keys, 2)
    good = torch.tensor([0, 3, 7], dtype=torch.int32, device=cuda)
    for k, ks in ((empty, bad), (empty, None), (keys, good)):
        out = fa.prompt_attention(empty, k, k, bad, kv_starts=ks, status=status.zero_())
        assert int(status) == N.DEV_LENGTH_RANGE and out.shape == (0, 2, 64)
    fa.prompt_attention(empty, empty, empty, none, kv_starts=bad, status=status.zero_())
    assert int(status) == N.DEV_LENGTH_RANGE
    for k, ks in ((empty, none), (keys, good)):
        fa.prompt_attention(empty, k, k, none, kv_starts=ks, workspace=ws[:fa.prompt_workspace(empty, k, k, 2).numel()],
                            status=status.zero_())
        assert int(status) == 0
    # the plan of the last call serves one like it
    fa.prompt_attention(empty, keys, keys, none, kv_starts=good, workspace=ws, plan_ready=True, status=status)
    assert int(status) == 0
    arena = pp.kv_cache.Int8KvArena.zeros(2, 2, 64, 16, cuda)
    arena.append_prompt(empty, empty, bad, none[:2], status=status.zero_())
    assert int(status) == N.DEV_LENGTH_RANGE
    arena.append_prompt(empty, empty, bad, none[:2])
    arena.append_prompt(empty, empty, none, none[:2], status=status.zero_())
    assert int(status) == 0 and not arena.k.any() and not arena.v_scale.any()


BAD_STATUS = [torch.empty(0, dtype=torch.int32), torch.zeros(1, dtype=torch.uint8), torch.zeros(1, dtype=torch.bfloat16),
              torch.zeros(1, dtype=torch.int64), torch.zeros(1)]


def test_status_words(pp):
    check, here = pp.int8_kv_ops.check_status, torch.device("cpu")
    check(None, here), check(torch.zeros(1, dtype=torch.int32), here), check(torch.zeros(3, dtype=torch.uint32), here)
    for bad in BAD_STATUS:
        with pytest.raises(pp.PreconditionError, match="status"):
            check(bad, here)
    with pytest.raises(pp.PreconditionError, match="status"):
        check(torch.zeros(1, dtype=torch.int32), torch.device("cuda", 0))


@pytest.mark.gpu
def test_status_words_are_checked(pp, cuda):
    """The kernels write 32 bits: into a smaller word's neighbours, or nowhere where there is no element."""
    x = torch.randn(4, 2, 64, device=cuda)
    starts = torch.tensor([0, 4], dtype=torch.int32, device=cuda)
    arena = pp.kv_cache.Int8KvArena.zeros(1, 2, 64, 16, cuda)
    for bad in [b.to(cuda) for b in BAD_STATUS] + [torch.zeros(1, dtype=torch.int32)]:
        with pytest.raises(pp.PreconditionError):
            pp.fused_attention.prompt_attention(x, x, x, starts, status=bad)
        with pytest.raises(pp.PreconditionError):
            pp.fused_attention.plan_prompt(x, x, x, starts, torch.empty(1 << 20, dtype=torch.uint8, device=cuda), status=bad)
        with pytest.raises(pp.PreconditionError):
            arena.append_prompt(x, x, starts, starts[:1], status=bad)
        with pytest.raises(pp.PreconditionError):
            pp.sampling.token_logprobs(x[:, 0], starts.repeat(2), status=bad)
