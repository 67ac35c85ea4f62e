"""Plans of packed prompts on the B200: which calls one that is kept in a workspace
serves, what the others do, batches of thousands of sequences, two at once."""
from __future__ import annotations

import pytest
import torch

from test_gpu_prompt import check, starts_of, tensors

pytestmark = pytest.mark.gpu

BOTH = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])


@BOTH
@pytest.mark.parametrize("other", ["causal", "max_ctas", "sequences", "queries", "keys", "heads", "kv_heads", "head_dim"])
def test_a_plan_of_another_geometry_is_refused(pp, cuda, other, dtype):
    """The workspace is large enough for every call here; the plan is cut along the keys."""
    fa = pp.fused_attention
    lens, kv_lens = [3, 200, 1], [3000, 1200, 5000]
    more = tensors(cuda, 205, 9201, 8, 2, 128, dtype, seed=9)  # a row that no sequence holds
    q, k, v = more[0][:204], more[1][:9200], more[2][:9200]
    qs, ks = starts_of(lens, cuda), starts_of(kv_lens, cuda)
    ws = torch.zeros(fa.prompt_workspace(q, k, v, 3).numel() * 2, dtype=torch.uint8, device=cuda)
    fa.plan_prompt(q, k, v, qs, ws, kv_starts=ks)
    plan = ws.clone()
    a = dict(q=q, k=k, v=v, q_starts=qs, kv_starts=ks)
    if other == "causal":
        a.update(causal=False)
    elif other == "max_ctas":
        a.update(max_ctas=7)
    elif other == "sequences":
        a.update(q_starts=qs[:3], kv_starts=ks[:3])
    elif other == "queries":
        a.update(q=more[0])
    elif other == "keys":
        a.update(k=more[1], v=more[2])
    elif other == "heads":
        a.update(q=q[:, :6])
    elif other == "kv_heads":
        a.update(k=k[:, :1], v=v[:, :1])
    else:
        a.update(q=q[..., :64], k=k[..., :64], v=v[..., :64])
    out = torch.full_like(a["q"], 7.0, memory_format=torch.contiguous_format)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    fa.prompt_attention(**a, workspace=ws, plan_ready=True, out=out, status=status)
    assert int(status) == pp._native.DEV_PLAN_MISMATCH and (out == 7).all()
    assert torch.equal(ws, plan)
    fa.prompt_attention(**a, workspace=ws, plan_ready=True, out=out)  # without a status word too
    assert (out == 7).all()
    # the plan is as good as before, and a call that makes its own replaces it
    check(fa.prompt_attention(q, k, v, qs, kv_starts=ks, workspace=ws, plan_ready=True, status=status.zero_()),
          q, k, v, lens, kv_lens, True)
    assert int(status) == 0
    fa.prompt_attention(**a, workspace=ws, out=out, status=status)
    assert int(status) == 0 and not (out[:203] == 7).all(-1).any()


@BOTH
@pytest.mark.parametrize("fill", [0, 1, 255])
def test_a_workspace_without_a_plan_is_refused(pp, cuda, fill, dtype):
    q, k, v = tensors(cuda, 300, 3000, 4, 2, 64, dtype)
    fa = pp.fused_attention
    qs, ks = starts_of([300], cuda), starts_of([3000], cuda)
    ws = fa.prompt_workspace(q, k, v, 1).fill_(fill)
    out, status = torch.full_like(q, 7.0), torch.zeros(1, dtype=torch.int32, device=cuda)
    fa.prompt_attention(q, k, v, qs, kv_starts=ks, workspace=ws, plan_ready=True, out=out, status=status)
    assert int(status) == pp._native.DEV_PLAN_MISMATCH and (out == 7).all() and (ws == fill).all()
    assert "plan" in pp._native.status_message(int(status))


def test_a_plan_is_void_after_a_call_that_gave_up(pp, cuda):
    """Such a call leaves the counter of its list somewhere in the list (word 1 of the workspace) and clears the last
    word of the geometry (word 7): later calls write nothing, instead of a part of their rows, until the next plan."""
    q, k, v = tensors(cuda, 300, 3000, 4, 2, 64, torch.bfloat16)
    fa = pp.fused_attention
    qs, ks = starts_of([300], cuda), starts_of([3000], cuda)
    ws = fa.prompt_workspace(q, k, v, 1)
    fa.plan_prompt(q, k, v, qs, ws, kv_starts=ks)
    header = ws[:32].view(torch.int32)
    assert int(header[0]) > 1 and int(header[1]) == 0 and int(header[7]) != 0
    header[1], header[7] = 1, 0
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    for _ in range(2):
        out = torch.full_like(q, 7.0)
        fa.prompt_attention(q, k, v, qs, kv_starts=ks, workspace=ws, plan_ready=True, out=out, status=status.zero_())
        assert int(status) == pp._native.DEV_PLAN_MISMATCH and (out == 7).all()
    fa.plan_prompt(q, k, v, qs, ws, kv_starts=ks)
    fa.prompt_attention(q, k, v, qs, kv_starts=ks, workspace=ws, plan_ready=True, out=out, status=status.zero_())
    assert int(status) == 0
    check(out, q, k, v, [300], [3000], True)


@BOTH
def test_a_plan_serves_other_strides_and_types(pp, cuda, dtype):
    """The work list depends on shapes and lengths alone."""
    fa = pp.fused_attention
    q, k, v = tensors(cuda, 150, 2000, 4, 4, 64, torch.float32)
    qs, ks = starts_of([100, 50], cuda), starts_of([1500, 500], cuda)
    ws = fa.prompt_workspace(q, k, v, 2)
    fa.plan_prompt(q, k, v, qs, ws, kv_starts=ks)
    q, k, v = (t.to(dtype).transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = fa.prompt_attention(q, k, v, qs, kv_starts=ks, workspace=ws, plan_ready=True, status=status)
    check(out, q, k, v, [100, 50], [1500, 500], True)
    assert int(status) == 0


@pytest.mark.parametrize("sequences", [2047, 2048, 2049, 5000])
def test_thousands_of_sequences(pp, cuda, sequences):
    """On both sides of 2048, beyond which the plan keeps the sequences' first entries in the workspace; one of them
    long, and empty ones throughout and at the end."""
    lens = [(i * 7919) % 5 for i in range(sequences)]
    lens[sequences // 3] = 1000
    lens[-3:] = [0, 0, 0]
    n = sum(lens)
    q, k, v = tensors(cuda, n + 2, n + 2, 2, 1, 64, torch.bfloat16, seed=2)
    out = torch.full_like(q, 7.0)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    starts = starts_of(lens, cuda)
    pp.fused_attention.prompt_attention(q, k, v, starts, out=out, status=status)
    assert int(status) == 0 and (out[n:] == 7).all() and out.isfinite().all()
    at = starts.tolist()
    for s in sorted({*range(0, sequences, 41), sequences // 3, sequences - 4}):
        a, b = at[s], at[s + 1]
        check(out[a:b], q[a:b], k[a:b], v[a:b], [b - a], [b - a], True)
    bad = starts.clone()
    bad[-1] = n + 3
    pp.fused_attention.prompt_attention(q, k, v, bad, out=out.fill_(7), status=status)
    assert int(status) == pp._native.DEV_LENGTH_RANGE and (out == 7).all()


@BOTH
def test_cut_rows_on_two_streams(pp, cuda, dtype):
    """Calls whose rows are cut along the keys and merged, on two streams at once."""
    fa = pp.fused_attention
    lens, kv = [3, 1, 40], [6000, 3000, 2000]
    qs, ks = starts_of(lens, cuda), starts_of(kv, cuda)
    data = [tensors(cuda, 44, 11000, 8, 2, 128, dtype, seed=s) for s in (1, 2)]
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [[], []]
    torch.cuda.synchronize()
    for _ in range(6):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                outs[s].append(fa.prompt_attention(*data[s], qs, kv_starts=ks))
    torch.cuda.synchronize()
    for s in range(2):
        check(outs[s][0], *data[s], lens, kv, True)
        assert all(torch.equal(outs[s][0], o) for o in outs[s])
