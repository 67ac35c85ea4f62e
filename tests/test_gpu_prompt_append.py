"""Append of packed prompts into the int8 arena on the B200: codes and scales
bit for bit those of int8_kv_ops.quantize, in the slots the starts name."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_prompt import starts_of

pytestmark = pytest.mark.gpu


def near_ties(n, h, d, dev, dtype, seed):
    """Heavy-tailed rows, every third one on or next to half-integer quotients of its own scale."""
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    x = torch.randn(n, h, d, device=dev, generator=g) * torch.exp(2 * torch.randn(n, h, 1, device=dev, generator=g))
    top = x.abs().amax(-1, keepdim=True)
    scale = torch.maximum(top / 127, torch.tensor(1e-12, device=dev))
    codes = torch.randint(-127, 127, (n, h, d), device=dev, generator=g) + 0.5
    tie = codes * scale
    bits = tie.view(torch.int32) + torch.randint(-2, 3, (n, h, d), device=dev, generator=g, dtype=torch.int32)
    x[::3] = bits.view(torch.float32)[::3]
    x[::3, :, :1] = top[::3]
    return x.to(dtype)


def run(pp, dev, k, v, lens, offsets, capacity, first=0, starts=None):
    arena = pp.kv_cache.Int8KvArena.zeros(len(lens), k.shape[1], k.shape[2], capacity, dev)
    arena.k.fill_(99), arena.v.fill_(98), arena.k_scale.fill_(5), arena.v_scale.fill_(6)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    arena.append_prompt(k, v, starts_of(lens, dev, first) if starts is None else starts,
                        torch.tensor(offsets, dtype=torch.int32, device=dev), status=status)
    return arena, int(status)


def expected(pp, arena, k, v, lens, offsets, first=0):
    h, cap, d = arena.heads, arena.capacity, arena.head_dim
    want = []
    for x, fill, sfill in ((k, 99, 5.0), (v, 98, 6.0)):
        codes, scales = pp.int8_kv_ops.quantize(x.contiguous(), check_finite=False)
        c = torch.full((len(lens), h, cap, d), fill, dtype=torch.uint8, device=x.device)
        s = torch.full((len(lens), h, cap), sfill, device=x.device)
        t = first
        for b, (n, o) in enumerate(zip(lens, offsets)):
            keep = max(0, min(n, cap - o))
            c[b, :, o:o + keep] = codes[t:t + keep].transpose(0, 1)
            s[b, :, o:o + keep] = scales[t:t + keep].transpose(0, 1)
            t += n
        want.append((c.view(-1, cap, d), s.view(-1, cap)))
    return want


def same(arena, want):
    (k, ks), (v, vs) = want
    return torch.equal(arena.k, k) and torch.equal(arena.v, v) and torch.equal(arena.k_scale, ks) \
        and torch.equal(arena.v_scale, vs)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("lens,offsets,heads,d,capacity", [
    ([1], [0], 1, 64, 1),
    ([5], [3], 3, 128, 9),
    ([0, 17, 0, 64, 1], [4, 0, 2, 1, 30], 7, 64, 66),
    ([1023], [1], 24, 64, 1024),
    ([300, 511, 77], [0, 0, 100], 16, 128, 512),
    ([65, 129], [0, 7], 100, 64, 136),
    ([3] * 700, [0, 1] * 350, 2, 64, 5),
])
def test_codes_and_scales_are_the_quantizers(pp, cuda, lens, offsets, heads, d, capacity, dtype):
    n = sum(lens)
    k, v = near_ties(n, heads, d, cuda, dtype, 1), near_ties(n, heads, d, cuda, dtype, 2)
    arena, status = run(pp, cuda, k, v, lens, offsets, capacity)
    assert status == 0
    assert same(arena, expected(pp, arena, k, v, lens, offsets))


def test_equals_appending_token_by_token(pp, cuda):
    lens, h, d = [9, 4], 4, 128
    k, v = near_ties(13, h, d, cuda, torch.bfloat16, 3), near_ties(13, h, d, cuda, torch.bfloat16, 4)
    arena, _ = run(pp, cuda, k, v, lens, [2, 0], 16)
    other = pp.kv_cache.Int8KvArena.zeros(2, h, d, 16, cuda)
    other.k.fill_(99), other.v.fill_(98), other.k_scale.fill_(5), other.v_scale.fill_(6)
    for i in range(4):
        at = torch.tensor([2 + i, i], dtype=torch.int32, device=cuda)
        other.append(k[[i, 9 + i]].reshape(-1, d), v[[i, 9 + i]].reshape(-1, d), at)
    for i in range(6):
        assert torch.equal(arena.k[:h, i], other.k[:h, i]) and torch.equal(arena.v_scale[:h, i], other.v_scale[:h, i])
    assert torch.equal(arena.k[h:], other.k[h:]) and torch.equal(arena.v[h:], other.v[h:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_extremes(pp, cuda, dtype):
    """Zero rows (the scale's floor), the smallest and largest floats, NaN and infinities (reported)."""
    x = torch.randn(8, 2, 64, device=cuda)
    x[0] = 0
    x[1] = 1e-38 * x[1].sign()
    x[2] *= 1e-41
    x[3] = 3.0e38 * x[3].sign()
    x[4, 0] *= 1e-13
    x[5] *= 1e36
    x = x.to(dtype)
    arena, status = run(pp, cuda, x, -x, [8], [0], 8)
    assert status == 0 and same(arena, expected(pp, arena, x, -x, [8], [0]))
    x[6, 1, 5], x[7, 0, 63] = math.nan, math.inf
    arena, status = run(pp, cuda, x, -x, [8], [0], 8)
    assert status == pp._native.DEV_NONFINITE_INPUT and same(arena, expected(pp, arena, x, -x, [8], [0]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_views_and_odd_strides(pp, cuda, dtype):
    lens, h, d = [20, 50], 3, 64
    x = near_ties(70, 3 * h, d, cuda, dtype, 5).view(70, 3, h, d)
    for k, v in ((x[:, 1], x[:, 2]), (x.transpose(1, 2)[:, :, 0], x[:, 2])):
        arena, status = run(pp, cuda, k, v, lens, [1, 0], 64)
        assert status == 0 and same(arena, expected(pp, arena, k, v, lens, [1, 0]))
    flat = torch.empty(70, h * d + 3, dtype=dtype, device=cuda)
    odd = flat[:, 1:1 + h * d].unflatten(1, (h, d))
    odd.copy_(x[:, 0])
    arena, status = run(pp, cuda, odd, x[:, 1], lens, [1, 0], 64)
    assert status == 0 and same(arena, expected(pp, arena, odd, x[:, 1], lens, [1, 0]))


def test_slots_beyond_the_capacity_and_rows_of_no_sequence(pp, cuda):
    lens, h, d = [30, 20, 10], 2, 64
    k, v = (near_ties(80, h, d, cuda, torch.bfloat16, s) for s in (6, 7))
    offs = [0, 25, 2**31 - 1]
    arena, status = run(pp, cuda, k, v, lens, offs, 32, first=7)
    assert status == pp._native.DEV_OFFSET_RANGE
    assert same(arena, expected(pp, arena, k, v, lens, [0, 25, 32], first=7))


@pytest.mark.parametrize("starts", [[0, 30, 20, 40], [0, 10, 20, 81], [5, 4, 4, 4]])
def test_bad_starts_write_nothing(pp, cuda, starts):
    k, v = (near_ties(80, 2, 64, cuda, torch.bfloat16, s) for s in (6, 7))
    arena, status = run(pp, cuda, k, v, [0, 0, 0], [0, 0, 0], 64,
                        starts=torch.tensor(starts, dtype=torch.int32, device=cuda))
    assert status == pp._native.DEV_LENGTH_RANGE
    assert (arena.k == 99).all() and (arena.v == 98).all() and (arena.k_scale == 5).all() and (arena.v_scale == 6).all()


def test_captured_replay_takes_new_lengths(pp, cuda):
    k, v = (near_ties(60, 2, 128, cuda, torch.bfloat16, s) for s in (8, 9))
    arena = pp.kv_cache.Int8KvArena.zeros(2, 2, 128, 64, cuda)
    starts, offsets = starts_of([20, 40], cuda), torch.zeros(2, dtype=torch.int32, device=cuda)
    arena.append_prompt(k, v, starts, offsets)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        arena.append_prompt(k, v, starts, offsets)
    for lens, offs in (([20, 40], [0, 0]), ([60, 0], [4, 9]), ([1, 59], [63, 5])):
        arena.k.fill_(99), arena.v.fill_(98), arena.k_scale.fill_(5), arena.v_scale.fill_(6)
        starts.copy_(starts_of(lens, cuda)), offsets.copy_(torch.tensor(offs, device=cuda))
        graph.replay()
        assert same(arena, expected(pp, arena, k, v, lens, offs))


def test_every_mantissa_of_a_maximum(pp, cuda):
    """All 2^23 maxima between 1 and 2, each with 63 elements on or within two units of half-integer quotients."""
    n, d = 2**23, 64
    top = torch.arange(2**23, dtype=torch.int32, device=cuda).add_(0x3F800000).view(torch.float32)
    g = torch.Generator(device=cuda)
    g.manual_seed(12)
    x = torch.randint(-127, 127, (n, 1, d), device=cuda, generator=g).float().add_(0.5)
    x.mul_((top / torch.full_like(top, 127.0))[:, None, None])
    x.view(torch.int32).add_(torch.randint(-2, 3, (n, 1, d), device=cuda, generator=g, dtype=torch.int32))
    x.clamp_(min=-top[:, None, None], max=top[:, None, None])
    x[:, 0, 0] = top
    arena = pp.kv_cache.Int8KvArena.zeros(1, 1, d, n, cuda)
    arena.append_prompt(x, x, starts_of([n], cuda), torch.zeros(1, dtype=torch.int32, device=cuda))
    codes, scales = pp.int8_kv_ops.quantize(x.view(1, n, d))
    assert torch.equal(arena.k_scale, scales) and torch.equal(arena.k, codes) and torch.equal(arena.v, codes)
