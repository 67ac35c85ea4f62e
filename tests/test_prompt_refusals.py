"""What the prompt operators refuse, on the CPU: nothing here launches a
kernel.  The C entry points check their arguments before they look for a
device; the Python ones check tensors before they call the library."""
from __future__ import annotations

import ctypes as C

import pytest
import torch


def prompt(pp, **kw):
    N = pp._native
    base = dict(sequences=2, heads=4, kv_heads=2, head_dim=64, dtype=N.DTYPE_BF16, q_tokens=10, kv_tokens=10, causal=1,
                softmax_scale=0.0, flags=0, max_ctas=0, q_token_stride=256, q_head_stride=64, k_token_stride=128,
                k_head_stride=64, v_token_stride=128, v_head_stride=64, q=4096, k=8192, v=16384)
    base.update(kw)
    g = N.PpPrompt(struct_size=C.sizeof(N.PpPrompt))
    for name, value in base.items():
        setattr(g, name, value)
    return g


BAD_GEOMETRY = [
    dict(struct_size=8), dict(sequences=0), dict(heads=0), dict(kv_heads=0), dict(heads=5), dict(heads=65 * 2),
    dict(head_dim=96), dict(dtype=7), dict(q_tokens=2**31), dict(kv_tokens=2**32 - 1), dict(sequences=2**31),
    dict(softmax_scale=-1.0), dict(softmax_scale=float("inf")), dict(softmax_scale=float("nan")),
    dict(max_ctas=2**20),
]


@pytest.mark.parametrize("bad", BAD_GEOMETRY, ids=str)
def test_prompt_geometry(pp, bad):
    N = pp._native
    g = prompt(pp, **bad)
    args = (C.byref(g), 64, 64, 4096, 1 << 30, None, None)
    assert N.lib.pp_b200_plan_prompt(*args) == N.STATUS_PRECONDITION and N.last_error()
    assert N.lib.pp_b200_prompt_workspace_size(C.byref(g)) == 0
    assert N.lib.pp_b200_prompt_attention(C.byref(g), 64, 64, 4096, 4096, 1 << 30, None, None) == N.STATUS_PRECONDITION


@pytest.mark.parametrize("bad", [dict(q=0), dict(k=0), dict(v=0), dict(q=4097), dict(k=4099), dict(v=8193),
                                 dict(k_token_stride=2**40), dict(q_head_stride=2**36)], ids=str)
def test_prompt_tensors(pp, bad):
    N = pp._native
    g = prompt(pp, **bad)
    assert N.lib.pp_b200_prompt_attention(C.byref(g), 64, 64, 4096, 4096, 1 << 30, None, None) == N.STATUS_PRECONDITION
    assert "prompt_attention" in N.last_error()


def test_prompt_starts(pp):
    N = pp._native
    g = prompt(pp)
    for starts in ((0, 64), (66, 64), (64, 66)):
        assert N.lib.pp_b200_prompt_attention(C.byref(g), *starts, 4096, 4096, 1 << 30, None, None) == N.STATUS_PRECONDITION
    assert N.lib.pp_b200_plan_prompt(C.byref(g), 64, 64, 4096, 1 << 30, 2, None) == N.STATUS_PRECONDITION
    assert N.lib.pp_b200_plan_prompt(None, 64, 64, 4096, 1 << 30, None, None) == N.STATUS_PRECONDITION


def test_workspace_size_grows_with_the_batch_and_stays_bounded(pp):
    N = pp._native
    size = lambda **kw: N.lib.pp_b200_prompt_workspace_size(C.byref(prompt(pp, max_ctas=148, **kw)))  # noqa: E731
    one = size(sequences=1, q_tokens=1)
    assert 0 < one < size(sequences=1, q_tokens=100000) < size(sequences=1, q_tokens=10**7)
    assert size(sequences=10**6) > 10**6 * 48
    assert size(q_tokens=0, kv_tokens=0) > 0
    assert size(head_dim=128) > size(head_dim=64)


def append_args(pp, **kw):
    N = pp._native
    a = N.PpKvArena(C.sizeof(N.PpKvArena), 8, 4, 64, 128, 0, 4096, 4096, 4096, 4096)
    base = dict(arena=a, k=4096, v=4096, dtype=N.DTYPE_BF16, tokens=10, kt=256, kh=64, vt=256, vh=64, starts=64,
                offsets=64, status=None, stream=None)
    base.update(kw)
    return [C.byref(base["arena"])] + [base[n] for n in list(base)[1:]]


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(tokens=2**31), dict(kt=2**40), dict(starts=0), dict(starts=65),
                                 dict(offsets=0), dict(offsets=66), dict(status=3)], ids=str)
def test_append(pp, bad):
    N = pp._native
    assert N.lib.pp_b200_prompt_append(*append_args(pp, **bad)) == N.STATUS_PRECONDITION
    assert "prompt_append" in N.last_error()


def test_append_arena(pp):
    N = pp._native
    for field, value in (("rows", 0), ("heads", 3), ("head_dim", 96), ("capacity", 0), ("k", 0), ("k", 8), ("v_scale", 2),
                         ("struct_size", 4)):
        args = append_args(pp)
        a = N.PpKvArena(C.sizeof(N.PpKvArena), 8, 4, 64, 128, 0, 4096, 4096, 4096, 4096)
        setattr(a, field, value)
        args[0] = C.byref(a)
        assert N.lib.pp_b200_prompt_append(*args) == N.STATUS_PRECONDITION, field


@pytest.mark.parametrize("bad", [dict(dtype=5), dict(choices=0), dict(choices=2**31), dict(choices=2**31 - 1), dict(rows=2**31), dict(top=33),
                                 dict(stride=2**40)], ids=str)
def test_logprobs(pp, bad):
    N = pp._native
    a = dict(logits=4096, dtype=0, rows=4, choices=100, stride=100, targets=64, bounds=None, top=2, lp=64, ent=64,
             rank=64, ids=64, best=64, status=None, stream=None)
    a.update(bad)
    assert N.lib.pp_b200_token_logprobs(*a.values()) == N.STATUS_PRECONDITION
    assert "token logprobs" in N.last_error()


def test_python_refuses_before_the_library(pp):
    P = pp.PreconditionError
    fa, sampling = pp.fused_attention, pp.sampling
    q = torch.zeros(4, 2, 64)
    s = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(P):  # a CPU tensor
        fa.prompt_attention(q, q, q, s)
    with pytest.raises(P):
        fa.prompt_attention(q[0], q, q, s)
    for starts in (s.long(), s[:1], s.view(1, 2), torch.zeros(4, dtype=torch.int32)[::2]):
        with pytest.raises(P, match="starts"):
            fa.prompt_attention(q, q, q, starts)
    with pytest.raises(P, match="starts"):
        fa.prompt_attention(q, q, q, s, kv_starts=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(P):
        sampling.token_logprobs(torch.zeros(3, 5), torch.zeros(3, dtype=torch.int32))
    arena = pp.kv_cache.Int8KvArena.zeros(1, 2, 64, 8, "cpu")
    with pytest.raises(P):
        arena.append_prompt(q, q, s, s[:1])


def test_status_text(pp):
    assert "window" in pp._native.status_message(pp._native.DEV_WINDOW_RANGE)
