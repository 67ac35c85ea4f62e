"""Prompt operators of the int8-KV decoder, as cases to measure.

Three operators take a prompt through the decoder and score what it says:

  attend   fused_attention.prompt_attention: every token of a batch of packed
           prompts attends to its own sequence (causal or not, grouped heads,
           keys of earlier tokens ahead of the chunk, single tokens)
  append   Int8KvArena.append_prompt: the prompt's K/V quantized into the int8
           arena, then read back as bf16 the way a later chunk's prefill does
  score    sampling.token_logprobs: log probability and rank of given tokens,
           entropy and the best alternatives of each row of logits

Where `own` is false, `run` computes the same results with elementary torch
operations in f32; where it is true it calls the framework.
"""
import importlib
import random

import torch

own = False


# ------------------------------------------------------------------ the cases

def _attend(name, q_lens, heads, kv_heads, dim, dtype="bf16", causal=True, past="0"):
    """q_lens, past: lengths of the chunks and of the tokens before them, as
    comma-separated texts (one past for all, or one each)."""
    return {"name": name, "kind": "attend", "q_lens": q_lens, "past": past, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "causal": causal}


def _append(name, lens, heads, dim, dtype="bf16", offset=0):
    return {"name": name, "kind": "append", "lens": lens, "heads": heads, "dim": dim, "dtype": dtype, "offset": offset}


def _score(name, rows, choices, top, dtype="bf16", window=False):
    return {"name": name, "kind": "score", "rows": rows, "choices": choices, "top": top, "dtype": dtype,
            "window": window}


def listed():
    return [
        # a first stroke record or two before the first token is drawn: pure latency
        _attend("attend tiny", "17", 24, 24, 64),
        # the model's own shape with a full context of history to prefill
        _attend("attend one context", "1023", 24, 24, 64),
        # a batch of branches whose prompts differ in length, prefilled in one call
        _attend("attend ragged batch", "4096,1,733,2048,129,3011,64,1500", 16, 16, 128),
        # the longest prompt, with grouped heads
        _attend("attend long grouped", "16384", 16, 4, 128),
        # the next chunk of prompts that are already partly in the cache
        _attend("attend chunks", "256,255,300,17,512,128,200,33", 16, 16, 128, past="2048,1000,1,4000,513,0,3000,127"),
        # one new token for each of 32 sequences with grouped heads: reading the keys and values is all there is
        _attend("attend single tokens", ",".join(["1"] * 32), 16, 4, 128, past="4095"),
        # f32 model tensors, not causal
        _attend("attend f32", "300,511,77,1000", 24, 24, 64, dtype="f32", causal=False),
        # one prompt of a full context into the arena of the model's own shape
        _append("append one context", "1023", 24, 64, offset=1),
        # sixteen branches' prompts at the synthetic decoder's shape
        _append("append batch", ",".join(str(2048 - 37 * i) for i in range(16)), 16, 128),
        # the field heads of 256 primitives, each with its window of legal tokens
        _score("score field heads", 2304, 1024, 8, dtype="f32", window=True),
        # one decode step's logits over a large vocabulary
        _score("score one step", 8, 131072, 20),
        # every position of a prompt scored
        _score("score prompt", 4096, 32768, 5),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    kind = rng.choice(["attend"] * 4 + ["append"] * 2 + ["score"] * 3)
    if kind == "append":
        n, dim = log(1, 24), rng.choice([64, 128])
        longest = log(3, 2048)
        lens = ",".join(str(rng.randint(0 if n > 1 else 1, longest)) for _ in range(n - 1))
        lens = (lens + "," if lens else "") + str(longest)
        c = _append("", lens, rng.randint(1, 24), dim, rng.choice(["bf16", "bf16", "f32"]), rng.randint(0, 70))
    elif kind == "score":
        choices = log(3, 140000)
        rows = log(1, max(2, min(5000, 130_000_000 // choices)))
        c = _score("", rows, choices, rng.choice([0, 1, 5, 20, 32]), rng.choice(["bf16", "f32"]), rng.random() < 0.4)
    else:
        dim, group = rng.choice([64, 128]), rng.choice([1, 1, 2, 3, 4, 7, 8])
        kv_heads = rng.randint(1, max(1, min(8, 2048 // (dim * group))))
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        form = rng.choice(["prompts", "prompts", "chunks", "tokens"])
        n = log(1, 24)
        if form == "tokens":
            q, past = [1] * n, [log(1, 8192) for _ in range(n)]
        else:
            longest = log(2, 2048 if dtype == "f32" else 6000)
            while n > 1 and n * longest > 16000:  # the plain form pads every sequence to the longest
                n = n // 2
            q = [rng.randint(1, longest) for _ in range(n)]
            past = [0] * n if form == "prompts" else [log(1, 2500) for _ in range(n)]
        c = _attend("", ",".join(map(str, q)), kv_heads * group, kv_heads, dim, dtype, rng.random() < 0.8,
                    ",".join(map(str, past)))
    del c["name"]
    return c


def _numbers(text):
    return [int(x) for x in text.split(",")]


def _lengths(case):
    q = _numbers(case["q_lens"])
    past = _numbers(case["past"])
    past = past * len(q) if len(past) == 1 else past
    return q, [a + b for a, b in zip(q, past)]


def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


# --------------------------------------------------------------------- inputs

def _package():
    return importlib.import_module("pop2-bezier_b200")


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = _dtype(case)

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    def i32(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    s = {"case": case}
    if case["kind"] == "attend":
        q, kv = _lengths(case)
        s["max_q"], s["max_kv"] = max(q), max(kv)
        # q and k leave the decoder's RMS norm with unit variance, v the projection
        s["q"] = randn(sum(q), case["heads"], case["dim"]).to(dt)
        s["k"] = randn(sum(kv), case["kv_heads"], case["dim"]).to(dt)
        s["v"] = randn(sum(kv), case["kv_heads"], case["dim"]).to(dt)
        s["q_starts"], s["kv_starts"] = i32(_starts(q)), i32(_starts(kv))
    elif case["kind"] == "append":
        lens, h, d = _numbers(case["lens"]), case["heads"], case["dim"]
        s["capacity"] = max(lens) + case["offset"]
        s["k"], s["v"] = (randn(sum(lens), h, d) * 2).to(dt), randn(sum(lens), h, d).to(dt)
        s["starts"], s["offsets"] = i32(_starts(lens)), i32([case["offset"]] * len(lens))
        rows = len(lens) * h
        s["arena"] = [torch.zeros(rows, s["capacity"], d, dtype=torch.uint8, device=dev) for _ in range(2)] + \
                     [torch.zeros(rows, s["capacity"], dtype=torch.float32, device=dev) for _ in range(2)]
    else:
        n, c = case["rows"], case["choices"]
        s["logits"] = (randn(n, c) * 2.5).to(dt)
        start = torch.zeros(n, dtype=torch.int64, device=dev)
        count = torch.full((n,), c, dtype=torch.int64, device=dev)
        if case["window"]:
            count = torch.randint((c + 1) // 2, c + 1, (n,), device=dev, generator=g)
            start = (torch.rand(n, device=dev, generator=g) * (c - count + 1)).long()
            s["bounds"] = torch.stack([start, count], 1).to(torch.int32)
        # half of the given tokens are likely ones, as a prompt's are, half are anything
        x = s["logits"].float()
        at = torch.arange(c, device=dev)
        x = torch.where((at >= start[:, None]) & (at < (start + count)[:, None]), x, -torch.inf)
        likely = (x + 0.5 * randn(n, c)).argmax(1)
        anything = start + (torch.rand(n, device=dev, generator=g) * count).long().clamp(max=c - 1)
        s["targets"] = torch.where(torch.rand(n, device=dev, generator=g) < 0.5, likely, anything).to(torch.int32)
    return s


# ------------------------------------------------------------ the plain forms

def _plain_attend(s):
    """Every sequence padded to the longest one: softmax(q k' / sqrt(d)) v over
    the keys that a row sees; row i of a causal chunk of n tokens ahead of
    which p keys lie sees keys 0 .. p + i."""
    c = s["case"]
    qs, ks = s["q_starts"].long(), s["kv_starts"].long()
    nq, nk = qs[1:] - qs[:-1], ks[1:] - ks[:-1]
    dev = qs.device
    iq, ik = torch.arange(s["max_q"], device=dev), torch.arange(s["max_kv"], device=dev)
    live_q, live_k = iq < nq[:, None], ik < nk[:, None]
    at_q = (qs[:-1, None] + iq).clamp(max=s["q"].shape[0] - 1)
    at_k = (ks[:-1, None] + ik).clamp(max=s["k"].shape[0] - 1)
    b, h, hk, d = nq.numel(), c["heads"], c["kv_heads"], c["dim"]
    q = s["q"][at_q].float().view(b, s["max_q"], hk, h // hk, d).permute(0, 2, 3, 1, 4)  # b, hk, group, lq, d
    k = s["k"][at_k].float().permute(0, 2, 3, 1)  # b, hk, d, lk
    v = s["v"][at_k].float().permute(0, 2, 1, 3)
    scores = (q.reshape(b, hk, -1, d) @ k).view(b, hk, h // hk, s["max_q"], s["max_kv"]).mul_(d ** -0.5)
    seen = live_k[:, None, :].expand(b, s["max_q"], s["max_kv"])
    if c["causal"]:
        seen = seen & (ik <= (iq + (nk - nq)[:, None])[:, :, None])
    scores.masked_fill_(~seen[:, None, None], -torch.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp_()
    out = scores.view(b, hk, -1, s["max_kv"]) @ v / scores.sum(-1).view(b, hk, -1, 1)
    out = out.view(b, hk, h // hk, s["max_q"], d).permute(0, 3, 1, 2, 4).reshape(b, s["max_q"], h, d)
    return out[live_q].to(s["q"].dtype)


def _plain_append(s):
    """Per token and head: scale = max|x| / 127 (at least 1e-12), code = x /
    scale rounded to even; the arena read back as bf16(code * scale)."""
    starts, offsets = s["starts"].long(), s["offsets"].long()
    t = torch.arange(s["k"].shape[0], device=starts.device)
    branch = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    slot = offsets[branch] + t - starts[branch]
    b, h, d = starts.numel() - 1, s["case"]["heads"], s["case"]["dim"]

    def side(x):
        x = x.float()
        scale = (x.abs().amax(-1) / 127.0).clamp(min=1e-12)
        codes = torch.round(x / scale[..., None]).clamp(-127, 127)
        values = torch.zeros(b, h, s["capacity"], d, dtype=torch.bfloat16, device=x.device)
        scales = torch.zeros(b, h, s["capacity"], device=x.device)
        values[branch, :, slot] = (codes * scale[..., None]).to(torch.bfloat16)
        scales[branch, :, slot] = scale
        return values.view(b * h, -1, d), scales.view(b * h, -1)

    (k, ks), (v, vs) = side(s["k"]), side(s["v"])
    return {"k": k, "k_scale": ks, "v": v, "v_scale": vs}


def _plain_score(s):
    """Over the window of each row: lse = log(sum exp x); log p = x - lse;
    entropy = -sum p log p; rank = tokens ahead of the target in the order
    (larger logit, lower index), whose head is the list of alternatives."""
    c, x = s["case"], s["logits"].float()
    n = x.shape[1]
    at, target = torch.arange(n, device=x.device), s["targets"].long()[:, None]
    if c["window"]:
        lo, hi = s["bounds"][:, :1].long(), s["bounds"].long().sum(1, keepdim=True)
        x = torch.where((at >= lo) & (at < hi), x, -torch.inf)
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.double().sum(1, keepdim=True)
    lse = top.double() + torch.log(total)
    spread = torch.where(e > 0, e * (top - x), torch.zeros_like(e)).double().sum(1, keepdim=True)
    xt = x.gather(1, target)
    rank = ((x > xt) | ((x == xt) & (at < target))).sum(1)
    out = {"logprob": (xt.double() - lse).float()[:, 0], "entropy": (torch.log(total) + spread / total).float()[:, 0],
           "rank": rank.to(torch.int32)}
    if c["top"]:
        k = min(c["top"], n)
        best, ids = torch.sort(x, dim=1, descending=True, stable=True)
        out["top_ids"] = torch.full((x.shape[0], c["top"]), -1, dtype=torch.int32, device=x.device)
        out["top_logprobs"] = torch.full((x.shape[0], c["top"]), -torch.inf, device=x.device)
        inside = best[:, :k] > -torch.inf
        out["top_ids"][:, :k] = torch.where(inside, ids[:, :k], -1).to(torch.int32)
        out["top_logprobs"][:, :k] = (best[:, :k].double() - lse).float()
    return out


def run(state):
    s, kind = state, state["case"]["kind"]
    if not own:
        return _plain_attend(s) if kind == "attend" else _plain_append(s) if kind == "append" else _plain_score(s)
    pp = _package()
    if kind == "attend":
        return pp.fused_attention.prompt_attention(s["q"], s["k"], s["v"], s["q_starts"], kv_starts=s["kv_starts"],
                                                   causal=s["case"]["causal"])
    if kind == "append":
        arena = pp.kv_cache.Int8KvArena(*s["arena"], heads=s["case"]["heads"])
        arena.append_prompt(s["k"], s["v"], s["starts"], s["offsets"])
        return {"k": pp.int8_kv_ops.dequantize(arena.k, arena.k_scale, torch.bfloat16), "k_scale": arena.k_scale,
                "v": pp.int8_kv_ops.dequantize(arena.v, arena.v_scale, torch.bfloat16), "v_scale": arena.v_scale}
    r = pp.sampling.token_logprobs(s["logits"], s["targets"], top=s["case"]["top"], bounds=s.get("bounds"))
    out = {"logprob": r.logprob, "entropy": r.entropy, "rank": r.rank}
    if s["case"]["top"]:
        out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
    return out


# ------------------------------------------------------- what a pass has to do

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "attend":
        q, kv = _lengths(case)
        pairs = sum(n * (m - n) + n * (n + 1) // 2 if case["causal"] else n * m for n, m in zip(q, kv))
        moved = 2 * sum(q) * case["heads"] + 2 * sum(kv) * case["kv_heads"]
        return {"bytes": moved * case["dim"] * size, "flops": 4 * pairs * case["heads"] * case["dim"]}
    if case["kind"] == "append":
        lens = _numbers(case["lens"])
        tokens, slots = sum(lens) * case["heads"], len(lens) * case["heads"] * (max(lens) + case["offset"])
        return {"bytes": 2 * tokens * case["dim"] * size + 2 * slots * (case["dim"] * 2 + 4),
                "flops": 6 * tokens * case["dim"]}
    return {"bytes": case["rows"] * (case["choices"] * size + 16 + 8 * case["top"]),
            "flops": 6 * case["rows"] * case["choices"]}


# --------------------------------------------------------- 64-bit definitions

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attend":
        q_lens, kv_lens = _lengths(case)
        group = case["heads"] // case["kv_heads"]
        out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        q0 = k0 = 0
        for n, m in zip(q_lens, kv_lens):
            hidden = None
            if case["causal"]:
                hidden = torch.ones(n, m, dtype=torch.bool, device=out.device).triu(m - n + 1)
            for h in range(case["heads"]):
                k, v = s["k"][k0:k0 + m, h // group].double(), s["v"][k0:k0 + m, h // group].double()
                x = s["q"][q0:q0 + n, h].double() @ k.T / case["dim"] ** 0.5
                if hidden is not None:
                    x[hidden] = -float("inf")
                out[q0:q0 + n, h] = torch.softmax(x, -1) @ v
            q0, k0 = q0 + n, k0 + m
        return out
    if case["kind"] == "append":
        lens, h, d = _numbers(case["lens"]), case["heads"], case["dim"]
        got = {}
        for name in ("k", "v"):
            values = torch.zeros(len(lens), h, s["capacity"], d, dtype=torch.float64, device=s["k"].device)
            scales = torch.zeros(len(lens), h, s["capacity"], dtype=torch.float64, device=s["k"].device)
            t = 0
            for b, n in enumerate(lens):
                x = s[name][t:t + n].double().transpose(0, 1)
                sc = (x.abs().max(-1).values / 127).clamp(min=1e-12) if n else x.sum(-1)
                where = slice(case["offset"], case["offset"] + n)
                values[b, :, where] = (x / sc.unsqueeze(-1)).round().clamp(-127, 127) * sc.unsqueeze(-1)
                scales[b, :, where] = sc
                t += n
            got[name], got[name + "_scale"] = values.flatten(0, 1), scales.flatten(0, 1)
        return got
    logp = s["logits"].double()
    n, c = logp.shape
    if case["window"]:
        inside = torch.zeros(n, c + 1, device=logp.device)
        b = s["bounds"].long()
        inside.scatter_add_(1, b[:, :1], torch.ones(n, 1, device=logp.device))
        inside.scatter_add_(1, b.sum(1, keepdim=True), -torch.ones(n, 1, device=logp.device))
        logp = logp.masked_fill(inside.cumsum(1)[:, :c] < 0.5, -float("inf"))
    logp = torch.log_softmax(logp, 1)
    got = {"logprob": logp.gather(1, s["targets"].long()[:, None])[:, 0],
           "entropy": -torch.xlogy(logp.exp(), logp.exp()).sum(1), "rank": None}
    if case["top"]:
        best = torch.full((n, case["top"]), -float("inf"), dtype=torch.float64, device=logp.device)
        k = min(case["top"], c)
        best[:, :k] = logp.topk(k, 1).values
        got["top_ids"], got["top_logprobs"] = None, best
    return got


if __name__ == "__main__":  # the cases and what each has to move and compute
    for one in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(one.get("name", "-"), work(one))
