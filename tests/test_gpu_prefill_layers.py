"""Prefill through the decoder on the B200, layer by layer."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_prefill import small
from test_gpu_prompt import check

pytestmark = pytest.mark.gpu


def test_a_model_on_cuda_without_an_index_takes_prompts(pp, cuda):
    """torch.device("cuda") and the "cuda:0" that its tensors report are one device."""
    model, same = small(pp, "cuda", torch.bfloat16), small(pp, cuda, torch.bfloat16)
    x = torch.randn(13, 256, device=cuda).to(torch.bfloat16)
    out = model.prefill(x.clone(), [10, 0, 3])
    assert torch.equal(out, same.prefill(x.clone(), [10, 0, 3])) and int(model.status) == 0
    with pytest.raises(pp.PreconditionError):
        model.prefill(x.cpu(), [10, 0, 3])


def network(model, x, lengths, dtype):
    """The prompts' hidden states with elementary torch operations in `dtype`."""
    cfg, d, h = model.cfg, model.cfg.head_dim, model.cfg.heads

    def norm(t, w):
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w

    pos = torch.cat([torch.arange(n, device=x.device) for n in lengths])
    x = x.to(dtype)
    for L in model.layers:
        w = {name: t.to(dtype) for name, t in L.items()}
        qn, kn = w["rope"][:d], w["rope"][d:2 * d]
        cos, sin = (t[pos][:, None] for t in w["rope"][2 * d:].view(2, cfg.max_context, d // 2))
        q, k, v = (norm(x, w["norm1"]) @ w["qkv"].T).view(-1, 3, h, d).unbind(1)

        def turned(t):
            a, b = t[..., ::2], t[..., 1::2]
            return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)

        q, k = turned(norm(q, qn)), turned(norm(k, kn))
        rows, t = [], 0
        for n in lengths:
            s = (q[t:t + n].transpose(0, 1) @ k[t:t + n].permute(1, 2, 0)) / math.sqrt(d)
            e = torch.exp((s - s.amax(-1, keepdim=True)) if n else s)
            e = e * torch.ones(n, n, dtype=dtype, device=x.device).tril()
            rows.append((e / e.sum(-1, keepdim=True) @ v[t:t + n].transpose(0, 1)).transpose(0, 1))
            t += n
        x = x + torch.cat(rows).reshape(-1, h * d) @ w["proj"].T
        gate, up = (norm(x, w["norm2"]) @ w["gate_up"].T).chunk(2, 1)
        x = x + gate / (1 + torch.exp(-gate)) * up @ w["down"].T
    return norm(x, model.final_norm.to(dtype))


LENGTHS = [[150, 1, 77], [0, 200, 3], [1100, 0, 900]]  # the last is cut along the keys and merged


def deep(pp, dev, dtype):
    cfg = pp.decoder.DecoderConfig(layers=4, width=256, heads=4, head_dim=64, ffn_hidden=512, max_context=1200)
    return pp.decoder.SyntheticDecoder(cfg, 3, 1200, dev, seed=5, dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_every_layers_attention(pp, cuda, lengths, dtype):
    """Each layer's attention, over one plan, within the formula's bounds from that layer's own q, k and v."""
    model = deep(pp, cuda, dtype)
    x = torch.randn(sum(lengths), 256, device=cuda).to(dtype)
    seen = []

    def probe(layer, q, k, v, arena, att):
        check(att, q, k, v, lengths, lengths, True)
        seen.append(layer)

    model.prefill(x, lengths, probe=probe)
    assert seen == [0, 1, 2, 3] and int(model.status) == 0


@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_f32_prefill_is_as_exact_as_elementary_operations(pp, cuda, lengths):
    """Row by row against 64 bits.  The elementary f32 network and the decoder round the same operations; the sums'
    orders and the exponentials and roots differ, which leaves the bounds of both within a factor of 2, and a row's error
    lies within a factor of 4 of another's of the same length: 8 times the elementary network's worst row.  (A key too many
    or too few in a row moves it by more than 10^-3, a thousand times that.)"""
    model = deep(pp, cuda, torch.float32)
    g = torch.Generator(device=cuda)
    g.manual_seed(3)
    x = torch.randn(sum(lengths), 256, device=cuda, generator=g)
    want = network(model, x, lengths, torch.float64)

    def errors(t):
        return (t.double() - want).norm(dim=1) / want.norm(dim=1)

    limit = 8 * float(errors(network(model, x, lengths, torch.float32)).max())
    assert limit < 1e-4
    got = errors(model.prefill(x.clone(), lengths))
    assert float(got.max()) <= limit, (float(got.max()), limit)
