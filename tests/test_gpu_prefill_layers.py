"""Prefill through the decoder on the B200, layer by layer."""
from __future__ import annotations

import pytest
import torch

from test_gpu_prefill import small

pytestmark = pytest.mark.gpu


def test_a_model_on_cuda_without_an_index_takes_prompts(pp, cuda):
    """torch.device("cuda") and the "cuda:0" that its tensors report are one device."""
    model, same = small(pp, "cuda", torch.bfloat16), small(pp, cuda, torch.bfloat16)
    x = torch.randn(13, 256, device=cuda).to(torch.bfloat16)
    out = model.prefill(x.clone(), [10, 0, 3])
    assert torch.equal(out, same.prefill(x.clone(), [10, 0, 3])) and int(model.status) == 0
    with pytest.raises(pp.PreconditionError):
        model.prefill(x.cpu(), [10, 0, 3])
