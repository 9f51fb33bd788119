"""Prompt and shared-prefix calls whose form and kernels the library chooses."""

from __future__ import annotations

import pytest
import torch

from prompt_cases import tables, weights

from latent_attn import MLAConfig
from latent_attn import functional as F

pytestmark = pytest.mark.gpu

ABSORBED = 3


def config(heads):
    return MLAConfig(5120, 512, 128, 64, heads, 128)


@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float32])
def test_queries_at_any_address(cuda, kv):
    """Packed float32 queries that begin at any element take the absorbed form's kernels of aligned ones: the same
    bits."""
    heads, L, n = 16, 96, 4
    g = torch.Generator().manual_seed(3)
    cache = torch.randn(2, L, 576, generator=g).to(kv).to(cuda)
    W_UK, W_UV = (w.to(cuda) for w in weights(heads, kv, 4))
    cos, sin = (t.to(cuda) for t in tables(L))
    q_nope, q_rope = (torch.randn(2 * n, heads, d, generator=g).to(cuda) for d in (128, 64))
    run = lambda a, b: F.mla_prefill(cache, a, b, W_UK, W_UV, cos, sin, config(heads), kernel_variant=ABSORBED)
    want = run(q_nope, q_rope)

    def moved(t):
        b = torch.zeros(t.numel() + 1, device=cuda)
        b[1:] = t.flatten()
        return b[1:].view_as(t)

    for a, b in ((moved(q_nope), q_rope), (q_nope, moved(q_rope)), (moved(q_nope), moved(q_rope))):
        assert torch.equal(run(a, b), want)
