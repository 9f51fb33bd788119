"""mla_prefill's plain kernel with scores of 10^8 and more: the largest of a token's gets the whole weight."""

from __future__ import annotations

import pytest
import torch

from conftest import assert_close
from prompt_cases import as_double, reference, tables, weights

from latent_attn import MLAConfig
from latent_attn import functional as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("by", [1e9, 1e20, -1e20])
@pytest.mark.parametrize("heads,n", [(3, 5), (16, 33)])
def test_large_scores(cuda, by, heads, n):
    """Rope element 31 alone (which turns by 0.01 at most here) tells the rows apart, in steps larger than that does."""
    rows = 90
    g = torch.Generator().manual_seed(n)
    kv = torch.randn(2, rows, 576, generator=g)
    kv[..., 512:] = 0
    kv[..., 512 + 31] = -1 - torch.stack([torch.randperm(rows, generator=g) for _ in range(2)]) * 0.01
    kv = kv.bfloat16().to(cuda)
    q = torch.zeros(2 * n, heads, 192)
    q[..., 128 + 31] = by
    q = q.to(cuda)
    cfg = MLAConfig(5120, 512, 128, 64, heads, 128)
    W_UK, W_UV = (x.to(cuda) for x in weights(heads, torch.bfloat16, 3))
    cos, sin = (x.to(cuda) for x in tables(rows))
    out = F.mla_prefill(kv, q[..., :128], q[..., 128:], W_UK, W_UV, cos, sin, cfg, kernel_variant=1, out_dtype=torch.float32)
    qd = as_double(q)
    ref = reference([as_double(r) for r in kv], qd[..., :128], qd[..., 128:], as_double(W_UK), as_double(W_UV), as_double(cos),
                    as_double(sin), [n, n])[0]
    assert_close(out.double().cpu().numpy(), ref.numpy(), "f32", f"{by}")
