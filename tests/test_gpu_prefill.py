"""Prompts through the whole decoder on the B200: prefill, decode, scoring.

The reference here is the same network in 64 bits with PyTorch, from the
decoder's own weights."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_logprobs import exact, near

pytestmark = pytest.mark.gpu


def small(pp, dev, dtype, branches=3, capacity=200):
    cfg = pp.decoder.DecoderConfig(layers=2, width=256, heads=4, head_dim=64, ffn_hidden=512, max_context=256)
    return pp.decoder.SyntheticDecoder(cfg, branches, capacity, dev, seed=5, dtype=dtype)


def in_64_bits(model, x, lengths):
    cfg, d, h = model.cfg, model.cfg.head_dim, model.cfg.heads

    def norm(t, w):
        return t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w

    pos = torch.cat([torch.arange(n, device=x.device) for n in lengths])
    x = x.double()
    for L in model.layers:
        w = {k: v.double() for k, v in L.items()}
        qn, kn, tab = w["rope"][:d], w["rope"][d:2 * d], w["rope"][2 * d:].view(2, cfg.max_context, d // 2)
        cos, sin = tab[0][pos][:, None], tab[1][pos][:, None]
        q, k, v = (norm(x, w["norm1"]) @ w["qkv"].T).view(-1, 3, h, d).unbind(1)

        def rope(t):
            a, b = t[..., ::2], t[..., 1::2]
            return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)

        q, k = rope(norm(q, qn)), rope(norm(k, kn))
        outs, t = [], 0
        for n in lengths:
            s = torch.einsum("ihd,jhd->hij", q[t:t + n], k[t:t + n]) / math.sqrt(d)
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1), -math.inf)
            outs.append(torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v[t:t + n]))
            t += n
        x = x + torch.cat(outs).reshape(-1, h * d) @ w["proj"].T
        gate, up = (norm(x, w["norm2"]) @ w["gate_up"].T).chunk(2, 1)
        x = x + (torch.nn.functional.silu(gate) * up) @ w["down"].T
    return norm(x, model.final_norm.double())


def distance(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("lengths", [[150, 1, 77], [0, 200, 3], [128, 0, 0]])
def test_prefill_matches_the_network(pp, cuda, dtype, lengths):
    """A layer has about ten operations, each of which rounds its result (half a step relative) and sums up to 512
    products (at most 512 * 2^-24 relative to the sum of their sizes, about sqrt(512) times the result's): two layers
    stay within 20 * (half a step + 512 * sqrt(512) * 2^-24), doubled for the norms and the softmax between them."""
    model = small(pp, cuda, dtype)
    g = torch.Generator(device=cuda)
    g.manual_seed(2)
    x = torch.randn(sum(lengths), 256, device=cuda, generator=g).to(dtype)
    seen = []

    def probe(layer, q, k, v, arena, att):
        codes, scales = pp.int8_kv_ops.quantize(k)
        vcodes, vscales = pp.int8_kv_ops.quantize(v)
        t = 0
        for b, n in enumerate(lengths):
            rows = slice(b * 4, b * 4 + 4)
            assert torch.equal(arena.k[rows, :n], codes[t:t + n].transpose(0, 1))
            assert torch.equal(arena.k_scale[rows, :n], scales[t:t + n].transpose(0, 1))
            assert torch.equal(arena.v[rows, :n], vcodes[t:t + n].transpose(0, 1))
            assert torch.equal(arena.v_scale[rows, :n], vscales[t:t + n].transpose(0, 1))
            assert not arena.k[rows, n:].any() and not arena.v_scale[rows, n:].any()
            t += n
        seen.append(layer)

    out = model.prefill(x.clone(), lengths, probe=probe)
    assert seen == [0, 1] and int(model.status) == 0
    half = torch.finfo(dtype).eps / 2
    assert distance(out, in_64_bits(model, x, lengths)) <= 40 * (half + 512 * math.sqrt(512) * 2.0**-24)


def test_decoding_goes_on_from_a_prefill(pp, cuda):
    """The next token by step() on the prefilled arenas against a prefill that is one token longer: they differ by the
    history's int8 codes, at most half a code of 127, 2^-8 of a row's largest element, in K and in V."""
    lengths = [90, 5, 140]
    model, longer = small(pp, cuda, torch.float32), small(pp, cuda, torch.float32)
    g = torch.Generator(device=cuda)
    g.manual_seed(4)
    parts = [torch.randn(n + 1, 256, device=cuda, generator=g) for n in lengths]
    model.prefill(torch.cat([p[:-1] for p in parts]), lengths)
    past = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    out = model.step(torch.stack([p[-1] for p in parts]), past)
    want = longer.prefill(torch.cat(parts), [n + 1 for n in lengths])
    last = torch.tensor(lengths, device=cuda).add(1).cumsum(0) - 1
    assert int(model.status) == 0 and int(longer.status) == 0
    # two layers, K and V each: 4 * 2^-8 of the largest element of 64, under four times a row's root mean square
    assert distance(out, want[last]) <= 16 * 2.0**-8
    assert torch.equal(model.arenas[0].k[:4, 90], longer.arenas[0].k[:4, 90])


def test_scoring_a_prefilled_prompt(pp, cuda):
    """Teacher-forced scores of a prompt's own next tokens, as a comparison of two models reads them."""
    lengths = [60, 33, 100]
    model = small(pp, cuda, torch.bfloat16)
    g = torch.Generator(device=cuda)
    g.manual_seed(8)
    embed = torch.randn(777, 256, device=cuda, generator=g).to(torch.bfloat16)
    tokens = torch.randint(0, 777, (sum(lengths),), device=cuda, generator=g, dtype=torch.int32)
    hidden = model.prefill(embed[tokens.long()], lengths)
    logits = hidden @ embed.T
    targets = torch.roll(tokens, -1)
    ends = torch.tensor(lengths, device=cuda).cumsum(0) - 1
    targets[ends] = -1  # nothing follows
    r = pp.sampling.token_logprobs(logits, targets.contiguous(), top=5)
    want = exact(logits.double(), targets, None, 5)  # a random model's tied head is nearly certain of its own token
    live = targets >= 0
    assert (r.logprob[~live] == -math.inf).all() and (r.rank[~live] == 777).all()
    near(r.logprob, want["lp"], want["err_lse"])
    near(r.entropy, want["ent"], want["err_ent"])
    near(r.top_logprobs, want["best"], want["err_lse"][:, None])
    assert torch.equal(r.top_ids.long(), want["ids"]) and torch.equal(r.rank.long(), want["rank"])


def test_prefill_refusals(pp, cuda):
    model = small(pp, cuda, torch.bfloat16)
    x = torch.zeros(10, 256, dtype=torch.bfloat16, device=cuda)
    for bad, lengths in ((x, [5, 5]), (x, [5, 4, 0]), (x, [201, 0, 0]), (x, [11, -1, 0]), (x.float(), [10, 0, 0]),
                         (x[:, :128], [10, 0, 0]), (x.cpu(), [10, 0, 0])):
        with pytest.raises(pp.PreconditionError):
            model.prefill(bad, lengths)
    assert model.prefill(x[:0], [0, 0, 0]).shape == (0, 256)
