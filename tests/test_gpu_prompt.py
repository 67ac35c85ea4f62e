"""Attention of packed prompts on the B200, against the formula in 64 bits.

Bounds.  With p the exact softmax row, A = sum_j p_j |v_j| and o the exact
output, a kernel that computes in f32 differs from o by at most
  E = A * (2 (ds + 2^-22 S) + (n + d) 2^-24 + 2^-20)
where ds = (d + 4) 2^-24 max_j scale sum |q_i k_ij| bounds the rounding of a
score (f32 sum of d products, the scale), S = max |score| log2(e) the rounding
of its shift and scale, each of which moves exp by as much relatively (once in
the numerator, once in the sum), (n + d) 2^-24 the sums over n keys, and 2^-20
the exponential itself and up to eight rescalings.  bf16 adds half a step,
2^-8, of every p_j (p is rounded for the matrix product: 2^-8 A) and half a
step of the result (2^-8 (|o| + all of the above))."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def starts_of(lens, dev, first=0):
    out = [first]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device=dev)


def exact_rows(q, k, v, causal, scale):
    """One sequence: q [n, h, d], k, v [m, hk, d] -> the result and its bound, both f64 [n, h, d]."""
    n, h, d = q.shape
    m, hk = k.shape[:2]
    bf = q.dtype == torch.bfloat16
    q, k, v = (t.double().transpose(0, 1) for t in (q, k, v))
    k, v = (t.repeat_interleave(h // hk, 0) for t in (k, v))
    s = q @ k.transpose(1, 2) * scale
    size = (q.abs() @ k.abs().transpose(1, 2) * scale)
    hidden = torch.zeros(n, m, dtype=torch.bool, device=q.device)
    if causal:
        hidden = torch.ones(n, m, dtype=torch.bool, device=q.device).triu(m - n + 1)
    s = s.masked_fill(hidden, -math.inf)
    size = size.masked_fill(hidden, 0)
    p = torch.softmax(s, -1)  # NaN where a row sees nothing
    seen = (~hidden).double()
    # a value that no row sees contributes nothing, whatever it holds
    clean = torch.nan_to_num(v, 0, 0, 0)
    spoiled = (seen @ (v != v).double()) > 0
    o = p.nan_to_num() @ clean
    a = p.nan_to_num() @ clean.abs()
    o = torch.where(spoiled | (seen.sum(-1) == 0)[None, :, None], torch.nan, o)
    if m:
        ds = (d + 4) * 2.0**-24 * size.amax(-1, keepdim=True)
        big = s.masked_fill(hidden, 0).abs().amax(-1, keepdim=True) * 1.4427
    else:
        ds = big = torch.zeros(h, n, 1, dtype=torch.float64, device=q.device)
    err = a * (2 * (ds + 2.0**-22 * big) + (m + d) * 2.0**-24 + 2.0**-20)
    if bf:
        err = err + 2.0**-8 * a
        err = err + 2.0**-8 * (o.nan_to_num().abs() + err)
    return o.transpose(0, 1), err.transpose(0, 1) + 1e-30


def check(out, q, k, v, q_lens, kv_lens, causal, scale=None, q_first=0, k_first=0):
    scale = scale or q.shape[2] ** -0.5
    q0, k0 = q_first, k_first
    for n, m in zip(q_lens, kv_lens):
        want, err = exact_rows(q[q0:q0 + n], k[k0:k0 + m], v[k0:k0 + m], causal, scale)
        got = out[q0:q0 + n].double()
        assert torch.equal(got.isnan(), want.isnan()), (n, m)
        bad = ((got - want).abs() > err).nan_to_num() & ~want.isnan()
        assert not bad.any(), (n, m, int(bad.sum()), float(((got - want).abs() / err).nan_to_num().max()))
        q0, k0 = q0 + n, k0 + m


def tensors(dev, q_tokens, kv_tokens, heads, kv_heads, d, dtype, seed=0, spread=1.0):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def r(*shape):
        return (torch.randn(*shape, device=dev, generator=g) * spread).to(dtype)

    return r(q_tokens, heads, d), r(kv_tokens, kv_heads, d), r(kv_tokens, kv_heads, d)


SHAPES = [
    # q_lens, past, heads, kv_heads
    ([1], [0], 1, 1),
    ([17], [0], 3, 3),
    ([127, 128, 129], [0, 0, 0], 4, 4),
    ([255, 256, 257, 1], [0, 0, 0, 0], 2, 2),
    ([0, 64, 0, 700, 0], [0, 0, 0, 0, 0], 4, 2),
    ([300], [0], 6, 2),
    ([130, 5], [0, 0], 7, 1),
    ([33, 1], [500, 129], 64, 1),
    ([1, 1, 1, 1], [0, 1, 127, 4000], 8, 2),
    ([1], [9000], 4, 1),
    ([100, 3, 260], [1, 1000, 127], 3, 3),
    ([1000], [1100], 2, 1),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}+{s[1]}x{s[2]}/{s[3]}")
def test_matches_the_formula(pp, cuda, shape, causal, d, dtype):
    q_lens, past, heads, kv_heads = shape
    kv_lens = [a + b for a, b in zip(q_lens, past)]
    q, k, v = tensors(cuda, sum(q_lens), sum(kv_lens), heads, kv_heads, d, dtype, seed=len(q_lens))
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = pp.fused_attention.prompt_attention(q, k, v, starts_of(q_lens, cuda), kv_starts=starts_of(kv_lens, cuda),
                                              causal=causal, status=status)
    check(out, q, k, v, q_lens, kv_lens, causal)
    assert int(status) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_default_keys_scale_and_peaked_scores(pp, cuda, dtype):
    """Without kv_starts the keys are the queries' tokens; large scores make the running maximum move often."""
    lens = [200, 1, 413]
    q, k, v = tensors(cuda, 614, 614, 4, 4, 64, dtype, seed=3, spread=4.0)
    k = (k.float() * torch.linspace(0.1, 3.0, 614, device=cuda)[:, None, None]).to(dtype)
    out = pp.fused_attention.prompt_attention(q, k, v, starts_of(lens, cuda), softmax_scale=0.2)
    check(out, q, k, v, lens, lens, True, scale=0.2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_that_see_no_key_are_nan(pp, cuda, d, dtype):
    """Fewer keys than queries: the first rows of a causal sequence see nothing; no keys at all: no row does."""
    q_lens, kv_lens = [300, 40, 7, 128], [120, 0, 7, 1]
    q, k, v = tensors(cuda, sum(q_lens), sum(kv_lens), 4, 2, d, dtype)
    for causal in (True, False):
        out = pp.fused_attention.prompt_attention(q, k, v, starts_of(q_lens, cuda), kv_starts=starts_of(kv_lens, cuda),
                                                  causal=causal)
        check(out, q, k, v, q_lens, kv_lens, causal)
    none = torch.empty(0, 2, d, dtype=dtype, device=cuda)
    out = pp.fused_attention.prompt_attention(q[:40], none, none, starts_of([40], cuda), kv_starts=starts_of([0], cuda))
    assert out.isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
def test_values_in_masked_places_do_not_matter(pp, cuda, d, dtype):
    """NaN and infinities in the keys and values of later tokens, of other sequences and behind the last one reach no
    row that does not see them, and every row that does."""
    q_lens, kv_lens = [150, 90, 200], [150, 300, 200]
    q, k, v = tensors(cuda, 440, 700, 4, 2, d, dtype, seed=5)
    for t, value in ((140, math.nan), (449, math.inf), (520, -math.inf), (650, math.nan)):
        v[t, :, ::3] = value
    k[600, 1] = math.nan
    k[651:] = math.inf
    out = pp.fused_attention.prompt_attention(q, k, v, starts_of(q_lens, cuda), kv_starts=starts_of(kv_lens, cuda))
    # what rows that see an infinite value or key hold is not defined beyond being not finite
    q0 = k0 = 0
    for n, m in zip(q_lens, kv_lens):
        qs, ks, vs = q[q0:q0 + n], k[k0:k0 + m], v[k0:k0 + m]
        see = torch.arange(m, device=cuda)[None] <= torch.arange(n, device=cuda)[:, None] + m - n
        spoiled_v = (see.double() @ (~vs.isfinite()).double().view(m, -1) > 0).view(n, 2, d).repeat_interleave(2, 1)
        spoiled_k = (see.double() @ (~ks.isfinite()).any(-1).double() > 0).repeat_interleave(2, 1)[..., None]
        fine = ~(spoiled_v | spoiled_k)
        got = out[q0:q0 + n]
        want, err = exact_rows(qs, ks.nan_to_num(0, 0, 0), vs.nan_to_num(0, 0, 0), True, d ** -0.5)
        assert ((got.double() - want).abs() <= err)[fine].all()
        assert not got.isfinite()[~fine].any()
        q0, k0 = q0 + n, k0 + m


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("layout", ["projection", "planes", "odd", "expanded"])
def test_views_and_strides(pp, cuda, layout, dtype):
    """Slices of a QKV projection, [heads, tokens, d] planes, rows off the 16-byte grid, a K/V head seen by expand."""
    lens, d, h = [70, 0, 190], 64, 4
    n = sum(lens)
    hk = h
    if layout == "projection":
        x = tensors(cuda, n, 1, 3 * h, 1, d, dtype)[0].view(n, 3, h, d)
        q, k, v = x[:, 0], x[:, 1], x[:, 2]
    elif layout == "planes":
        q, k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in tensors(cuda, n, n, h, h, d, dtype))
    elif layout == "odd":
        x = tensors(cuda, n, 1, 1, 1, 3 * h * d + 7, dtype)[0].view(n, -1)[:, 3:]
        q, k, v = (x[:, i * h * d:(i + 1) * h * d].unflatten(1, (h, d)) for i in range(3))
        assert k.data_ptr() % 16
    else:
        q, k, v = tensors(cuda, n, n, h, 1, d, dtype)
        k, v, hk = k.expand(n, 2, d), v.expand(n, 2, d), 2
    out = pp.fused_attention.prompt_attention(q, k, v, starts_of(lens, cuda))
    assert k.shape[1] == hk
    check(out, q, k, v, lens, lens, True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_rows_of_no_sequence_are_left_as_they_were(pp, cuda, dtype):
    lens = [130, 33]
    q, k, v = tensors(cuda, 400, 400, 2, 2, 128, dtype)
    out = torch.full_like(q, 7.0)
    pp.fused_attention.prompt_attention(q, k, v, starts_of(lens, cuda, first=10), out=out)
    assert (out[:10] == 7).all() and (out[173:] == 7).all()
    check(out, q, k, v, lens, lens, True, q_first=10, k_first=10)


@pytest.mark.parametrize("starts", [[0, 50, 40, 60], [0, 20, 101], [90, 80], [0, 2**31 - 1]])
def test_bad_starts_write_nothing_and_set_the_status(pp, cuda, starts):
    q, k, v = tensors(cuda, 100, 100, 2, 2, 64, torch.bfloat16)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = torch.full_like(q, 7.0)
    bad = torch.tensor(starts, dtype=torch.int32, device=cuda)
    good = torch.linspace(0, 100, len(starts), device=cuda).to(torch.int32)
    for qs, ks in ((bad, bad), (bad, good), (good, bad)):
        status.zero_()
        pp.fused_attention.prompt_attention(q, k, v, qs, kv_starts=ks, status=status, out=out)
        assert int(status) == pp._native.DEV_LENGTH_RANGE
        assert (out == 7).all()
    pp.fused_attention.prompt_attention(q, k, v, good, status=status.zero_(), out=out)
    assert int(status) == 0 and not (out == 7).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("max_ctas", [1, 5, 0])
def test_cut_and_whole_plans_agree_and_repeat_bit_for_bit(pp, cuda, dtype, max_ctas):
    """The same call twice gives the same bits, however the rows are cut along the keys and whoever finishes last."""
    q_lens, kv_lens = [3, 200, 1], [3000, 1200, 5000]
    q, k, v = tensors(cuda, 204, 9200, 8, 2, 128, dtype, seed=9)
    fa = pp.fused_attention
    ws = fa.prompt_workspace(q, k, v, 3, max_ctas=max_ctas)
    qs, ks = starts_of(q_lens, cuda), starts_of(kv_lens, cuda)
    fa.plan_prompt(q, k, v, qs, ws, kv_starts=ks, max_ctas=max_ctas)
    out = [fa.prompt_attention(q, k, v, qs, kv_starts=ks, workspace=ws, plan_ready=True, max_ctas=max_ctas)
           for _ in range(4)]
    check(out[0], q, k, v, q_lens, kv_lens, True)
    assert all(torch.equal(out[0], o) for o in out[1:])
    # the plan serves other tensors of the same shapes (the next layer)
    q2, k2, v2 = tensors(cuda, 204, 9200, 8, 2, 128, dtype, seed=10)
    o2 = fa.prompt_attention(q2, k2, v2, qs, kv_starts=ks, workspace=ws, plan_ready=True, max_ctas=max_ctas)
    check(o2, q2, k2, v2, q_lens, kv_lens, True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("past", [900, 1500, 20000])
def test_rows_cut_into_pieces(pp, cuda, past, d, dtype):
    """Few rows over many keys: two to more than eight pieces, tiles with rows that do not exist, a value that is
    not finite and that only the last tokens see."""
    q_lens = [50, 1, 90, 7]
    kv_lens = [50 + past, 1 + past // 2, 90 + past // 3, 7]
    q, k, v = tensors(cuda, sum(q_lens), sum(kv_lens), 6, 2, d, dtype, seed=past)
    v[sum(kv_lens[:1]) - 2] = math.nan
    v[sum(kv_lens[:3]) - 1, 0] = math.inf
    v[sum(kv_lens[:3]) - 1, 0, 3] = math.nan
    out = pp.fused_attention.prompt_attention(q, k, v, starts_of(q_lens, cuda), kv_starts=starts_of(kv_lens, cuda))
    at_q, at_k = 0, 0
    for n, m in zip(q_lens, kv_lens):
        rows, keys = slice(at_q, at_q + n), slice(at_k, at_k + m)
        want, err = exact_rows(q[rows], k[keys], v[keys].masked_fill(v[keys].isinf(), 0.0), True, d**-0.5)
        # the channels of K/V head 0 that the last token sees as inf
        inf = torch.zeros(n, 2, d, dtype=torch.bool, device=cuda)
        inf[n - 1] = v[keys][m - 1].isinf()
        inf = inf.repeat_interleave(3, 1)
        got = out[rows].double()
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.isinf(), inf & ~want.isnan())
        plain = ~inf & ~want.isnan()
        assert not (((got - want).abs() > err) & plain).any()
        at_q, at_k = at_q + n, at_k + m


@pytest.mark.parametrize("sequences", [1500, 40])
def test_many_short_sequences(pp, cuda, sequences):
    """More sequences than the plan's threads, most of them shorter than a tile."""
    lens = [(i * 7919) % 60 for i in range(sequences)]
    n = sum(lens)
    q, k, v = tensors(cuda, n, n, 2, 1, 64, torch.bfloat16, seed=2)
    out = pp.fused_attention.prompt_attention(q, k, v, starts_of(lens, cuda))
    at = starts_of(lens, cuda).tolist()
    for s in range(0, sequences, 37):
        a, b = at[s], at[s + 1]
        check(out[a:b], q[a:b], k[a:b], v[a:b], [b - a], [b - a], True)
    assert out.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_captured_graph_and_two_streams(pp, cuda, dtype):
    """A captured call replays on new inputs and lengths; calls on two streams with a workspace each do not meet."""
    fa = pp.fused_attention
    q, k, v = tensors(cuda, 300, 300, 4, 2, 128, dtype)
    lens = starts_of([100, 200], cuda)
    fa.prompt_attention(q, k, v, lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fa.prompt_attention(q, k, v, lens)
    for seed, cut in ((1, [100, 200]), (2, [299, 1]), (3, [0, 300])):
        a, b, c = tensors(cuda, 300, 300, 4, 2, 128, dtype, seed=seed)
        q.copy_(a), k.copy_(b), v.copy_(c), lens.copy_(starts_of(cut, cuda))
        graph.replay()
        check(out, q, k, v, cut, cut, True)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    data = [tensors(cuda, 700, 700, 4, 4, 64, dtype, seed=s) for s in (7, 8)]
    starts = starts_of([700], cuda)
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                outs[s].append(fa.prompt_attention(*data[s], starts))
    torch.cuda.synchronize()
    for s in range(2):
        check(outs[s][0], *data[s], [700], [700], True)
        assert all(torch.equal(outs[s][0], o) for o in outs[s])


def test_keys_behind_the_32_bit_border(pp, cuda):
    """Element offsets of keys beyond 2^32 (a cache of 17 GB)."""
    tokens = 2**32 // (16 * 128) + 5000
    k = torch.zeros(tokens, 16, 128, dtype=torch.bfloat16, device=cuda)
    g = torch.Generator(device=cuda)
    g.manual_seed(1)
    k[-3000:] = torch.randn(3000, 16, 128, device=cuda, generator=g).to(torch.bfloat16)
    q = torch.randn(40, 16, 128, device=cuda, generator=g).to(torch.bfloat16)
    ks = torch.tensor([tokens - 2900, tokens - 100], dtype=torch.int32, device=cuda)
    out = pp.fused_attention.prompt_attention(q, k, k, starts_of([40], cuda), kv_starts=ks)
    check(out, q, k[-2900:-100], k[-2900:-100], [40], [2800], True)
