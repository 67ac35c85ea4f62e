"""Scores of given tokens on the B200, against the formula in 64 bits.

Bounds.  Let s be the sum of e_i = exp(x_i - m) without the largest.  Each e_i
carries the exponential's own error (2^-21 relative), that of its argument
(|x_i - m| 2^-22: the difference, the change of base) and one more of each for
every time the running maximum moves (at most 40 of them with the merges of
threads, warps and pieces), and the sum has n terms added in chains of at most
n / 32 + 64.  So s is off by at most
  r = 41 * 2^-21 + 2^-22 a + (n / 32 + 64) 2^-24       relatively,
a = sum e_i |x_i - m| / s, which moves log1p(s) by at most r s / (1 + s) and
d / (1 + s) by 2 r times itself.  The result is rounded to f32 (2^-24).  An e_i
below 2^-126, the least normal f32, may count as 0: n of them move s, and so
log1p(s), by less than n 2^-126, and d, with |x_i - m| < 2^8 where e_i >= 2^-300
and nothing to speak of below, by less than n 2^-118."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def exact(x, targets, bounds, top):
    """x f64 [n, c] -> dict of f64 results, bounds of their errors, and the order's whole numbers."""
    n, c = x.shape
    dev = x.device
    at = torch.arange(c, device=dev)
    lo = torch.zeros(n, 1, dtype=torch.long, device=dev) if bounds is None else bounds[:, :1].long()
    hi = lo + (c if bounds is None else bounds[:, 1:].long())
    inside = (at >= lo) & (at < hi)
    xw = x.masked_fill(~inside, -math.inf)
    # log p = (x - m) - log1p(s): x - logsumexp(x) would lose a nearly certain token's digits even in 64 bits
    m = xw.amax(1, keepdim=True)
    e = torch.where(xw > -math.inf, (xw - m).exp(), torch.zeros_like(xw))
    e.scatter_(1, xw.argmax(1, keepdim=True), 0)
    gap = torch.where(e > 0, m - xw, torch.zeros_like(e))
    s, d = e.sum(1), (e * gap).sum(1)
    tail = torch.log1p(s)[:, None]
    ent = tail[:, 0] + d / (1 + s)
    r = 41 * 2.0**-21 + 2.0**-22 * (d / s.clamp(min=1e-300)) + (c / 32 + 64) * 2.0**-24
    err_lse = r * s / (1 + s) + c * 2.0**-126
    t = targets.long()[:, None]
    ok = (t >= lo) & (t < hi)
    tc = t.clamp(0, c - 1)
    xt = torch.where(ok, x.gather(1, tc), torch.full_like(m, -math.inf))
    lp = torch.where(ok, xt - m - tail, torch.full_like(m, -math.inf))[:, 0]
    rank = torch.where(ok, inside & ((x > xt) | ((x == xt) & (at < t))), inside).sum(1)
    order = torch.sort(xw, dim=1, descending=True, stable=True)
    k = min(top, c)
    ids = torch.full((n, top), -1, device=dev)
    best = torch.full((n, top), -math.inf, dtype=torch.float64, device=dev)
    listed = order.values[:, :k] > -math.inf
    ids[:, :k] = torch.where(listed, order.indices[:, :k], -1)
    best[:, :k] = torch.where(listed, order.values[:, :k] - m - tail, -math.inf)
    return dict(lp=lp, ent=ent, rank=rank, ids=ids, best=best, err_lse=err_lse,
                err_ent=err_lse + 2 * r * d / (1 + s) + c * 2.0**-118)


def near(got, want, err):
    got = got.double()
    want = torch.where(want < -torch.finfo(torch.float32).max, -math.inf, want)  # as f32 rounds it
    fin = want.isfinite()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[~fin].nan_to_num(7, 8, 9), want[~fin].nan_to_num(7, 8, 9))
    off = (got - want).abs()[fin]
    lim = (err + 2.0**-24 * want.abs())[fin]
    assert (off <= lim).all(), float((off / lim).max())


def check(pp, logits, targets, top, bounds=None):
    status = torch.zeros(1, dtype=torch.int32, device=logits.device)
    r = pp.sampling.token_logprobs(logits, targets, top=top, bounds=bounds, status=status)
    w = exact(logits.double(), targets, bounds, top)
    assert torch.equal(r.rank.long(), w["rank"])
    near(r.logprob, w["lp"], w["err_lse"])
    near(r.entropy, w["ent"], w["err_ent"])
    if top:
        assert torch.equal(r.top_ids.long(), w["ids"])
        near(r.top_logprobs, w["best"], w["err_lse"][:, None])
    else:
        assert r.top_ids is None and r.top_logprobs is None
    assert int(status) == 0
    return r


def make(dev, rows, choices, dtype, seed, spread=2.5):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    x = (torch.randn(rows, choices, device=dev, generator=g) * spread).to(dtype)
    t = torch.randint(0, choices, (rows,), device=dev, generator=g, dtype=torch.int32)
    best = x.float().argmax(1).int()
    return x, torch.where(torch.arange(rows, device=dev) % 2 == 0, best, t)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,choices,top", [
    (1, 1, 1), (3, 2, 5), (2, 31, 32), (5, 33, 0), (7, 255, 8), (4, 1024, 20), (300, 1000, 3), (2, 2049, 32),
    (1, 8191, 20), (3, 8193, 7), (40, 16384, 1), (1, 131072, 20), (9, 50001, 32), (600, 4099, 5), (2, 300007, 10),
])
def test_matches_the_formula(pp, cuda, rows, choices, top, dtype):
    x, t = make(cuda, rows, choices, dtype, rows + choices)
    check(pp, x, t, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("choices", [1, 7, 1024, 20000])
def test_windows(pp, cuda, choices, dtype):
    """Windows of every size from one column, at odd starts; targets inside, outside and none."""
    rows = 64
    x, t = make(cuda, rows, choices, dtype, 5)
    g = torch.Generator(device=cuda)
    g.manual_seed(6)
    count = torch.randint(1, choices + 1, (rows,), device=cuda, generator=g)
    count[:8] = 1
    start = (torch.rand(rows, device=cuda, generator=g) * (choices - count + 1)).long().clamp(max=choices - 1)
    bounds = torch.stack([start, count], 1).int()
    # what lies outside the window does not matter
    at = torch.arange(choices, device=cuda)
    outside = (at < start[:, None]) | (at >= (start + count)[:, None])
    x = torch.where(outside, torch.nan, x.float()).to(dtype)
    t[::5] = (start + count)[::5].int()  # just behind the window
    t[1] = -1
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    r = pp.sampling.token_logprobs(x, t, top=9, bounds=bounds, status=status)
    w = exact(torch.where(outside, 0.0, x.double()), t, bounds, 9)
    assert torch.equal(r.rank.long(), w["rank"]) and torch.equal(r.top_ids.long(), w["ids"])
    near(r.logprob, w["lp"], w["err_lse"])
    near(r.entropy, w["ent"], w["err_ent"])
    assert int(status) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("choices", [500, 9000, 70000])
def test_ties_go_to_the_lower_column(pp, cuda, choices, dtype):
    """Few distinct values, among them both zeros; whole rows of one value; a rising and a falling row."""
    g = torch.Generator(device=cuda)
    g.manual_seed(1)
    x = torch.randint(-2, 3, (8, choices), device=cuda, generator=g).float() * 0.5
    x = torch.where((x == 0) & (torch.rand(8, choices, device=cuda, generator=g) < 0.5), -0.0, x)
    x[1] = 3.25
    x[2] = -0.0
    x[3] = torch.arange(choices, device=cuda) / 64
    x[4] = -torch.arange(choices, device=cuda) / 64
    t = torch.tensor([0, choices - 1, 17, 5, 6, 100, 200, 300], dtype=torch.int32, device=cuda)
    check(pp, x.to(dtype), t, 32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,choices", [(3, 140001), (200, 40000), (40, 3000)])
@pytest.mark.parametrize("top", [1, 5, 32])
def test_rows_in_order(pp, cuda, top, rows, choices, dtype):
    """Rising, falling and half-sorted rows: every column, or none, is a candidate when it comes."""
    x, t = make(cuda, rows, choices, dtype, choices + top)
    x[0::3] = x[0::3].sort(1).values
    x[1::3] = x[1::3].sort(1, descending=True).values
    x[2::3, choices // 2:] = x[2::3, choices // 2:].sort(1).values
    check(pp, x, t, top)


def test_a_nearly_certain_token_keeps_its_digits(pp, cuda):
    """logprob about -1e-9: 1 + s would round it to 0 in f32."""
    x = torch.zeros(4, 1000, device=cuda)
    x[:, 123] = torch.tensor([20.0, 27.0, 40.0, 88.0], device=cuda)
    t = torch.full((4,), 123, dtype=torch.int32, device=cuda)
    r = check(pp, x, t, 2)
    assert (r.logprob[:3] < 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("choices", [300, 40000])
def test_infinities_and_nan(pp, cuda, choices, dtype):
    x, t = make(cuda, 8, choices, dtype, 3)
    x[0, ::2] = -math.inf
    x[1, :] = -math.inf
    x[1, 7] = 0.5
    x[2, :] = torch.finfo(dtype).min
    x[2, 11] = torch.finfo(dtype).max
    t[0], t[1], t[2] = 2, 7, 0
    check(pp, x[:3].contiguous(), t[:3].contiguous(), 5)
    x[3, :] = -math.inf  # nothing left
    x[4, 5] = math.nan
    x[5, 9] = math.inf
    x[6, :] = math.nan
    x[7, 0] = math.nan
    x[7, 1:] = -math.inf
    t[4] = 5
    r = pp.sampling.token_logprobs(x[3:].contiguous(), t[3:].contiguous(), top=4)
    assert r.logprob.isnan().all() and r.entropy.isnan().all()
    assert (r.top_ids[0] == -1).all() and (r.top_logprobs[0] == -math.inf).all()
    clean = x[4].float().nan_to_num(-1e30)
    assert torch.equal(r.top_ids[1].long(), torch.sort(clean, descending=True, stable=True).indices[:4])
    assert r.top_logprobs[1].isnan().all()
    assert int(r.rank[1]) == choices - 1  # a NaN target comes behind everything else
    assert int(r.top_ids[2, 0]) == 9
    assert (r.top_ids[3] == -1).all() and (r.top_ids[4] == -1).all()


def test_bad_and_empty_windows(pp, cuda):
    x, t = make(cuda, 5, 100, torch.float32, 4)
    bounds = torch.tensor([[0, 100], [90, 11], [50, 0], [101, 0], [2**31 - 1, 2**31 - 1]], dtype=torch.int32, device=cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    r = pp.sampling.token_logprobs(x, t, top=3, bounds=bounds, status=status)
    assert int(status) == pp._native.DEV_WINDOW_RANGE
    assert r.logprob[0].isfinite() and r.logprob[1:].isnan().all() and r.entropy[1:].isnan().all()
    assert (r.top_ids[1:] == -1).all() and (r.rank[1:] == 0).all()
    status.zero_()
    pp.sampling.token_logprobs(x[:3].contiguous(), t[:3].contiguous(), bounds=bounds[[0, 2, 2]].contiguous(), status=status)
    assert int(status) == 0  # an empty window is no error


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_strided_rows_and_odd_alignment(pp, cuda, dtype):
    big, t = make(cuda, 6, 3001, dtype, 8)
    for view in (big[:, 1:2000], big[:, 3:], big[1::2, :2999]):
        n = view.shape[0]
        tt = t[:n] % view.shape[1]
        check(pp, view, tt.int().contiguous(), 6)
    rows = big[:1].expand(4, 3001)  # one row seen four times
    check(pp, rows, t[:4].contiguous(), 6)


def test_no_rows_replay_and_repeat(pp, cuda):
    x, t = make(cuda, 4, 60000, torch.bfloat16, 9)
    r = pp.sampling.token_logprobs(x[:0], t[:0], top=3)
    assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 3)
    first = pp.sampling.token_logprobs(x, t, top=20)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = pp.sampling.token_logprobs(x, t, top=20)
    for _ in range(3):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(first, r))
    y, u = make(cuda, 4, 60000, torch.bfloat16, 10)
    x.copy_(y), t.copy_(u)
    graph.replay()
    w = exact(x.double(), t, None, 20)
    assert torch.equal(r.top_ids.long(), w["ids"]) and torch.equal(r.rank.long(), w["rank"])
