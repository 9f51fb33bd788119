"""A speculating server whose caches have a budget: trees drafted, a path of each accepted, rows weighed, caches cut back, in
turn, against rows and weights kept beside it."""

from __future__ import annotations

import pytest
import torch

from draft_cases import tree
from prompt_cases import tables, weights

from latent_attn import MLAConfig
from latent_attn import functional as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("block", [0, 64])
@pytest.mark.parametrize("each", [False, True])
def test_drafts_under_a_budget(cuda, block, each):
    """each: the tokens of every accepted path weigh the rows, a call per sequence; else the newest token of all of them."""
    heads, B, n, cap, keep = 16, 3, 10, 192, 70
    cfg = MLAConfig(5120, 512, 128, 64, heads, 128)
    g = torch.Generator().manual_seed(11)
    W_UK, W_UV = (x.to(cuda) for x in weights(heads, torch.bfloat16, 2))
    cos, sin = (x.to(cuda) for x in tables(cap))
    kw = {}
    if block:
        kw = {"block_table": torch.randperm(B * cap // block, generator=g).int().view(B, -1).to(cuda), "block_size": block}
        kv = torch.zeros(B * cap, 576, dtype=torch.bfloat16, device=cuda)
    else:
        kv = torch.zeros(B, cap, 576, dtype=torch.bfloat16, device=cuda)
    lens, wts = torch.zeros(B, dtype=torch.int32, device=cuda), torch.zeros(B, cap, device=cuda)

    def rand(*shape):
        return torch.randn(*shape, generator=g).bfloat16().to(cuda)

    def append(count):
        new = rand(B, count, 576)
        F.append_kv(kv, lens, new[..., :512].contiguous(), new[..., 512:].contiguous(), cfg, **kw)
        return new

    rows = list(append(50))
    sums = [torch.zeros(50, device=cuda) for _ in range(B)]
    for step in range(6):
        parents = [tree(n, 10 * step + s) for s in range(B)]
        paths = []
        for s, p in enumerate(parents):
            path, j = [], n - 1 - s
            while j >= 0:
                path.insert(0, j)
                j = p[j]
            paths.append(path)
        new, q = append(n), rand(B * n, heads, 192)
        out = F.mla_decode_tree(kv, q[..., :128], q[..., 128:], W_UK, W_UV, cos, sin, cfg,
                                torch.tensor(parents, dtype=torch.int32, device=cuda), seq_lens=lens, rotate_q=True, **kw)
        assert out.isfinite().all()
        F.accept_kv(kv, lens, n, torch.tensor([(p + [-1] * n)[:n] for p in paths], dtype=torch.int32, device=cuda), cfg, **kw)
        for s, p in enumerate(paths):
            rows[s] = torch.cat([rows[s], new[s, p]])
            sums[s] = torch.cat([sums[s], torch.zeros(len(p), device=cuda)])

        def weigh(w, cache, tokens, **more):
            F.weigh_kv(w, cache, tokens[..., :128], tokens[..., 128:], W_UK, cos, sin, cfg, rotate_q=True, **more)

        taken = [q[[s * n + j for j in (p if each else p[-1:])]] for s, p in enumerate(paths)]
        if each:
            for s in range(B):
                part = {"block_table": kw["block_table"][s:s + 1], "block_size": block} if block else {}
                weigh(wts[s:s + 1], kv if block else kv[s:s + 1], taken[s], seq_lens=lens[s:s + 1], **part)
        else:
            weigh(wts, kv, torch.cat(taken), seq_lens=lens, **kw)
        for s in range(B):
            alone = sums[s][None].clone()
            weigh(alone, rows[s][None].contiguous(), taken[s])
            sums[s] = alone[0]
            L = len(rows[s])
            assert int(lens[s]) == L
            assert (wts[s, :L] - sums[s]).norm() <= 1e-5 * sums[s].norm() and (wts[s, L:] == 0).all()
            sums[s] = wts[s, :L].clone()  # (the last bits differ: the rows are chosen by those of the one)
        kept = F.evict_kv(kv, lens, wts, cfg, keep, first=4, last=20, **kw)
        for s in range(B):
            at = kept[s][kept[s] >= 0].long()
            rows[s], sums[s] = rows[s][at], sums[s][at]
            L = len(at)
            assert int(lens[s]) == L <= keep and torch.equal(wts[s, :L], sums[s]) and (wts[s, L:] == 0).all()
            places = kw["block_table"][s].long()[torch.arange(L, device=cuda) // block] * block + torch.arange(
                L, device=cuda) % block if block else torch.arange(L, device=cuda) + s * cap
            assert torch.equal(kv.view(-1, 576)[places], rows[s])
    assert all(len(r) == keep for r in rows)
