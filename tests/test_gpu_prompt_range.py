"""fp16 caches whose values pass fp16's range when a row is expanded (the row itself is finite): the tokens that do not see
it are left as they are, those that see it get nothing finite."""

from __future__ import annotations

import pytest
import torch

from prompt_cases import tables, weights

from latent_attn import MLAConfig
from latent_attn import functional as F

pytestmark = pytest.mark.gpu

EXPANDED = 2


def large_row(g):
    """60,000 times signs: a value is a sum of 512 products of it with weights of about 1 / sqrt(512), so normal with a
    deviation of 60,000, and one of the 128 values of a head passes 65,520 but for a chance of 0.73^128."""
    return torch.cat([60000.0 * (torch.randint(0, 2, (512,), generator=g) * 2 - 1), torch.zeros(64)])


@pytest.mark.parametrize("heads,rows", [(4, (150, 80)), (16, (150, 80)), (32, (150, 80)), (128, (150, 80)), (128, (40, 700))])
def test_a_value_past_the_range(cuda, heads, rows):
    """By the size of the call: gathered in the expansion's workgroups, one tile per workgroup, four."""
    cfg = MLAConfig(5120, 512, 128, 64, heads, 128)
    g = torch.Generator().manual_seed(heads)
    total = sum(rows)
    kv = torch.randn(total, 576, generator=g).half().to(cuda)
    W_UK, W_UV = (w.to(cuda) for w in weights(heads, torch.float16, 2))
    cos, sin = (t.to(cuda) for t in tables(max(rows)))
    q = torch.randn(total, heads, 192, generator=g).half().to(cuda)
    off = torch.tensor([0, rows[0], total], dtype=torch.int32, device=cuda)
    run = lambda: F.mla_prefill(kv, q[..., :128], q[..., 128:], W_UK, W_UV, cos, sin, cfg, q_offsets=off, seq_offsets=off,
                                rotate_q=True, kernel_variant=EXPANDED)
    want = run()
    assert torch.isfinite(want).all()
    bad = [(rows[0] * 2 // 3, rows[0]), (rows[0] + 67, total)]  # rows, and the ends of their sequences
    for at, _ in bad:
        kv[at] = large_row(g).half().to(cuda)
    got = run()
    seen = torch.zeros(total, dtype=torch.bool, device=cuda)
    for at, end in bad:
        seen[at:end] = True
    assert torch.equal(got[~seen], want[~seen])
    assert not torch.isfinite(got[seen]).all(-1).any()


@pytest.mark.parametrize("heads", [4, 128])
def test_an_expanded_prefix(cuda, heads):
    """Its values are held at the largest number; a step behind it, which sees every row, gets nothing finite."""
    cfg = MLAConfig(5120, 512, 128, 64, heads, 128)
    g = torch.Generator().manual_seed(heads)
    rows = torch.randn(400, 576, generator=g).half()
    W_UK, W_UV = (w.to(cuda) for w in weights(heads, torch.float16, 2))
    cos, sin = (t.to(cuda) for t in tables(420))
    clean = F.expand_prefix(rows.to(cuda), W_UK, W_UV, cos, sin, cfg)
    rows[333] = large_row(g).half()
    p = F.expand_prefix(rows.to(cuda), W_UK, W_UV, cos, sin, cfg)
    v, old = (x.v.reshape(-1, heads, 128) for x in (p, clean))
    others = torch.arange(v.shape[0], device=cuda) != 333
    assert torch.equal(v[others], old[others]) and v[333].abs().max() == 65504
    k, old = (torch.cat([x.k_nope.reshape(-1, heads * 128), x.k_rope.reshape(-1, 64)], 1) for x in (p, clean))
    assert torch.equal(k[others], old[others]) and k[333].isnan().any()
    q = torch.randn(2, heads, 192, generator=g).to(cuda)
    got = F.mla_decode_shared(p, torch.randn(2, 20, 576, generator=g).half().to(cuda), q[..., :128].contiguous(),
                              q[..., 128:].contiguous(), W_UK, W_UV, cos, sin, cfg, kernel_variant=EXPANDED)
    assert not torch.isfinite(got).all(-1).any()
