"""Scores of any size in mla_decode_tree and weigh_kv: the largest of them gets the whole weight where they are far apart. The
running maximum starts below every finite one."""

from __future__ import annotations

import pytest
import torch

from conftest import assert_close
from draft_cases import weight_places
from test_gpu_tree import Case as Tree
from test_gpu_weigh import Case as Weigh

pytestmark = pytest.mark.gpu


def rows_of(lengths, kv, seed):
    """Latents at random; of the rope part element 31 alone (which turns by 0.04 at most here), from -1 down to -1.9 in steps
    that the type and the rotation tell apart."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in lengths:
        r = torch.randn(n, 576, generator=g)
        r[:, 512:] = 0
        r[:, 512 + 31] = -1 - torch.randperm(n, generator=g) * 0.9 / n
        out.append(r.to(kv).float())
    return out


def queries(c, by):
    """Scores of -by and less (times some 0.1)."""
    c.q[..., :] = 0
    c.q[..., 128 + 31] = by
    return c


BY = [1e9, 1e20, -1e20, 1e34, -1e34]


@pytest.mark.parametrize("n,heads,lengths", [(7, 16, [30, 57]), (64, 128, [70, 64, 99]), (4, 3, [20, 60])])
@pytest.mark.parametrize("variant", [0, 1])
@pytest.mark.parametrize("by", BY)
def test_trees(cuda, n, heads, lengths, variant, by):
    c = queries(Tree(cuda, "paged", lengths, n, heads=heads, rotate_q=False, data=rows_of(lengths, torch.bfloat16, n)), by)
    got = c.run(kernel_variant=variant)
    assert_close(got.double().cpu().numpy(), c.reference().numpy(), "bf16", f"{n} {heads}")


@pytest.mark.parametrize("tokens,heads", [(1, 16), (3, 16), (2, 128), (3, 7)])
@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("by", BY)
def test_weights(cuda, tokens, heads, kv, variant, by):
    lengths = [90, 33, tokens]
    c = queries(Weigh(cuda, "paged", lengths, tokens, heads=heads, kv=kv, q=torch.float32, rotate_q=False,
                      data=rows_of(lengths, kv, tokens)), by)
    w = torch.zeros_like(c.weights)
    c.run(w, kernel_variant=variant)
    got = w.cpu().double().view(-1)
    for s, r in enumerate(c.reference()[0]):
        assert float(r.sum()) == heads * tokens and (r == r.round()).all()  # one row per token
        assert torch.equal(got[weight_places(c.layout, s, len(r))], r)


@pytest.mark.parametrize("tokens,heads", [(1, 16), (3, 16), (2, 128), (3, 7)])
@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("by", [1.0, 1e4, 1e9])
def test_large_scores_that_are_alike(cuda, tokens, heads, kv, variant, by):
    """Rows that are one and the same share a token's weight evenly, whatever their score: its sum is the number of rows that the
    token sees, which a maximum of 10^8 that it was added to as a logarithm would swallow."""
    lengths = [300, 33, tokens]
    g = torch.Generator().manual_seed(tokens)
    row = torch.randn(1, 576, generator=g).to(kv).float()
    row[:, 512:] = 0
    c = Weigh(cuda, "paged", lengths, tokens, heads=heads, kv=kv, q=torch.float32, rotate_q=False,
              data=[row.expand(n, -1).contiguous() for n in lengths])
    c.q *= by
    w = torch.zeros_like(c.weights)
    c.run(w, kernel_variant=variant)
    got = w.cpu().double().view(-1)
    for s, n in enumerate(lengths):
        sees = torch.arange(tokens) + n - tokens + 1
        want = torch.tensor([heads * float((1.0 / sees[sees > k]).sum()) for k in range(n)], dtype=torch.float64)
        off = (got[weight_places(c.layout, s, n)] - want).abs()
        # the exponentials are 1; a reciprocal, its sums over tokens and heads
        assert (off <= (tokens * heads + 4) * 2.0 ** -24 * want).all()
