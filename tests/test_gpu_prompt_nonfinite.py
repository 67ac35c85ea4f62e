"""Values that are not finite in the prompts on the B200: rows that see them, rows
that do not, and how long a call with them takes."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_prompt import check, exact_rows, starts_of, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (6, 2), (16, 1)])
@pytest.mark.parametrize("lens,past", [([700, 90, 3], [0, 0, 0]), ([300, 1, 40], [200, 1000, 77]), ([20, 1], [5000, 3000])])
def test_nan_reaches_the_rows_that_see_it_and_no_others(pp, cuda, lens, past, heads, kv_heads, d, dtype):
    """NaN in keys and in values, in one element, one channel of every token, at the ends and on both sides of a border
    of key tiles: a row is NaN where it sees one, and keeps its digits where it does not."""
    kv = [n + p for n, p in zip(lens, past)]
    for case in range(6):
        q, k, v = tensors(cuda, sum(lens), sum(kv), heads, kv_heads, d, dtype, seed=case)
        n = kv[0]
        if case == 0:
            k[5], v[5] = math.nan, math.nan
        elif case == 1:
            v[5, 0, 3] = math.nan
        elif case == 2:
            v[:, 0, d - 1] = math.nan
        elif case == 3:
            v[[n // 2 // 128 * 128, n // 2 // 128 * 128 + 127, n - 1], -1, 7] = math.nan
        elif case == 4:
            v[5, :, 3], v[n - 2, :, 40] = math.nan, math.nan  # one explained by a row's own keys, one not
        else:
            v[n - 30:n, 0] = math.nan
            k[n - 1] = math.nan
        out = pp.fused_attention.prompt_attention(q, k, v, starts_of(lens, cuda), kv_starts=starts_of(kv, cuda))
        q0 = k0 = 0
        for a, b in zip(lens, kv):
            ks, vs = k[k0:k0 + b], v[k0:k0 + b]
            see = torch.arange(b, device=cuda)[None] <= torch.arange(a, device=cuda)[:, None] + b - a
            group = heads // kv_heads
            bad = (see.double() @ ks.isnan().any(-1).double() > 0)[..., None] \
                | (see.double() @ vs.isnan().double().view(b, -1) > 0).view(a, kv_heads, d)
            bad = bad.repeat_interleave(group, 1)
            want, err = exact_rows(q[q0:q0 + a], ks.nan_to_num(0), vs.nan_to_num(0), True, d ** -0.5)
            got = out[q0:q0 + a].double()
            assert torch.equal(got.isnan(), bad), case
            assert ((got - want).abs() <= err)[~bad].all(), case
            q0, k0 = q0 + a, k0 + b


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
def test_infinite_values(pp, cuda, causal, d):
    """+inf and -inf in one channel each of a later sequence's tokens, in the same key tile: no row here sees them."""
    lens = [70, 100, 13]
    q, k, v = tensors(cuda, 183, 183, 4, 2, d, torch.bfloat16)
    v[170:, :, 0], v[170:, :, d - 1] = math.inf, -math.inf
    out = pp.fused_attention.prompt_attention(q, k, v, starts_of(lens, cuda), causal=causal)
    check(out[:170], q[:170], k[:170], v[:170], lens[:2], lens[:2], causal)
    assert not out[170:, :, [0, d - 1]].isfinite().any()
    check(out[170:, :, 1:d - 1], q[170:], k[170:], v[170:, :, 1:d - 1], lens[2:], lens[2:], causal, scale=d ** -0.5)


@pytest.mark.parametrize("where", ["a token", "an element", "a channel", "all keys", "cut"])
def test_a_call_with_nan_takes_about_as_long(pp, cuda, where):
    """A row whose own keys hold the NaN is not computed again.  When every such row was, the calls below took 400 to
    3000 times as long as without NaN; 20 is far from both."""
    n = 4096
    q, k, v = tensors(cuda, n, n, 16, 4, 128, torch.bfloat16)
    qs, ks = starts_of([n], cuda), None
    if where == "cut":
        q, qs, ks = q[:8], starts_of([8], cuda), starts_of([n], cuda)
    out = torch.empty_like(q)

    def run():
        times = []
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            pp.fused_attention.prompt_attention(q, k, v, qs, kv_starts=ks, out=out)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    clean = run()
    if where == "a token":
        q[5], k[5], v[5] = math.nan, math.nan, math.nan
    elif where == "all keys":
        k[:], v[:] = math.nan, math.nan
    elif where == "a channel":
        v[:, :, 3] = math.nan
    else:
        v[5, 0, 3] = math.nan
    assert run() < 20 * clean
    assert out[-1].isnan().any()
