"""A table whose rows overlap in memory (one row expanded, a sliding window) is
looked up like any other: the same bits as from a copy."""

from __future__ import annotations

import pytest
import torch

from graspo_amd import ops
from graspo_amd.embedding import token_embedding

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("H", [1, 7, 64])
def test_rows_that_overlap(H, dtype):
    V = 30
    flat = torch.randn(V + H, generator=torch.Generator().manual_seed(H)).to(dtype).cuda()
    ids = torch.arange(V, device="cuda").flip(0)
    for w in (flat[:H].expand(V, H), flat.as_strided((V, H), (1, 1)), flat[:1].expand(V, H)):
        plain = w.contiguous()
        want = ops.embedding(ids, plain, scale=3.0)[0]
        assert torch.equal(ops.embedding(ids, w, scale=3.0)[0], want)
        assert torch.equal(token_embedding(ids, w, scale=3.0), want)
        wd = w.detach().requires_grad_()
        out = token_embedding(ids, wd)
        (g,) = torch.autograd.grad(out, [wd], torch.ones_like(out))
        assert g.shape == (V, H) and bool((g == 1).all())
