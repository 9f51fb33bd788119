"""GPU tests of mla_decode_tree, accept_kv, weigh_kv and evict_kv over caches whose byte offsets pass 32 bits: one
sequence of 3.9 million rows, and sequences that begin behind 4 GiB."""

from __future__ import annotations

import pytest
import torch

from conftest import assert_close
from prompt_cases import weights

from latent_attn import MLAConfig
from latent_attn import functional as F

pytestmark = pytest.mark.gpu

HEADS, LONG, REGIONS = 16, 3_900_096, 48  # 1,152 bytes a row: 4.49e9, and 4.40e9 before the last region


@pytest.fixture(scope="module")
def long(cuda):
    g = torch.Generator(device=cuda).manual_seed(1)
    cfg = MLAConfig(5120, 512, 128, 64, HEADS, 128)
    kv = torch.randn(1, LONG, 576, generator=g, device=cuda, dtype=torch.bfloat16)
    q = torch.randn(4, HEADS, 192, generator=g, device=cuda).bfloat16()
    W_UK, W_UV = (x.to(cuda) for x in weights(HEADS, torch.bfloat16, 5, 512, 128, 128))
    angle = torch.rand(LONG, 32, generator=g, device=cuda) * 6.28
    yield cfg, kv, q, W_UK, W_UV, angle.cos(), angle.sin()
    del kv, angle
    torch.cuda.empty_cache()


def rotate(x, cos, sin):
    a, b = x[..., :32], x[..., 32:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def scores(kv, q, W_UK, cos, sin, q_at, k_at):
    """(tokens, heads, rows) float32 scores of packed rows, keys at positions k_at."""
    qa = torch.stack([q[:, h, :128].float() @ W_UK.view(HEADS, 128, 512)[h].float() for h in range(HEADS)], 1)
    qr = rotate(q[..., 128:].float(), cos[q_at][:, None], sin[q_at][:, None])
    full = torch.cat([qa, qr], -1).reshape(-1, 576)
    out = torch.empty(full.shape[0], kv.shape[0], device=kv.device)
    for i in range(0, kv.shape[0], 1 << 19):
        rows = kv[i:i + (1 << 19)].float()
        at = k_at[i:i + (1 << 19)]
        rows[:, 512:] = rotate(rows[:, 512:], cos[at], sin[at])
        out[:, i:i + (1 << 19)] = full @ rows.T
    return out.view(q.shape[0], HEADS, -1) * 192 ** -0.5


def test_a_long_sequence(cuda, long):
    cfg, kv, q, W_UK, W_UV, cos, sin = long
    lens = torch.tensor([LONG], dtype=torch.int32, device=cuda)
    parents = torch.tensor([[-1, 0, 0, 1]], dtype=torch.int32, device=cuda)
    depth, sees = torch.tensor([0, 1, 1, 2], device=cuda), torch.tensor([[0, 0], [0, 1], [0, 2], [0, 1]])
    at = LONG - 4 + depth
    k_at = torch.cat([torch.arange(LONG - 4, device=cuda), at])
    s = scores(kv[0], q, W_UK, cos, sin, at, k_at)
    for j in range(4):
        for i in range(4):
            if i != j and i not in sees[j].tolist():
                s[j, :, LONG - 4 + i] = -float("inf")
    s = s.double().softmax(-1)
    latent = sum((s[:, :, i:i + (1 << 19)].float().reshape(4 * HEADS, -1) @ kv[0, i:i + (1 << 19), :512].float())
                 for i in range(0, LONG, 1 << 19)).view(4, HEADS, 512)
    want = torch.stack([latent[:, h] @ W_UV.view(HEADS, 128, 512)[h].float().T.contiguous() for h in range(HEADS)], 1)
    got = F.mla_decode_tree(kv, q[..., :128], q[..., 128:], W_UK, W_UV, cos, sin, cfg, parents, seq_lens=lens, rotate_q=True)
    assert_close(got.double().cpu().numpy(), want.double().cpu().numpy(), "bf16")
    del s
    # one token's weights: fp32's worth of the softmax (the reference's products are fp32 sums of 576 terms: 2^-16)
    w = torch.zeros(1, LONG, device=cuda)
    F.weigh_kv(w, kv, q[:1, :, :128], q[:1, :, 128:], W_UK, cos, sin, cfg, seq_lens=lens, rotate_q=True)
    s = scores(kv[0], q[:1], W_UK, cos, sin, torch.tensor([LONG - 1], device=cuda), torch.arange(LONG, device=cuda))
    s = s[0].double().softmax(-1).sum(0)
    assert float((w[0].double() - s).norm() / s.norm()) <= 2.0 ** -14
    assert abs(float(w.double().sum()) - HEADS) <= 1e-4
    # the rows that stay, moved from both ends of the sequence
    own = kv.clone()
    kept = F.evict_kv(own, lens, w, cfg, 5000, first=4, last=1000)
    order = s[4:LONG - 1000].topk(3996).indices + 4
    assert int(lens) == 5000 and (kept[0, 1:] > kept[0, :-1]).all()
    assert kept[0, :4].tolist() == [0, 1, 2, 3] and kept[0, -1000:].tolist() == list(range(LONG - 1000, LONG))
    assert torch.isin(kept[0, 4:4000].long(), order).float().mean() > 0.99  # (neighbours in rank may change places)
    assert torch.equal(own[0, :5000], kv[0, kept[0].long()])
    # and an accepted path's, at the far end
    lens.fill_(LONG)
    own.copy_(kv)
    F.accept_kv(own, lens, 4, torch.tensor([[0, 2, 3, -1]], dtype=torch.int32, device=cuda), cfg)
    assert int(lens) == LONG - 1
    assert torch.equal(own[0, LONG - 4:LONG - 1], kv[0, [LONG - 4, LONG - 2, LONG - 1]])
    assert torch.equal(own[0, :LONG - 4], kv[0, :LONG - 4])


@pytest.mark.parametrize("paged", [False, True])
def test_sequences_behind_4_gib(cuda, long, paged):
    """The same few rows at the far end of a pool, or in the last of the regions, as in a small cache."""
    cfg, kv, q, W_UK, W_UV, cos, sin = long
    near = kv[0, :192].clone()
    parents = torch.tensor([[-1, 0, 0, 1]], dtype=torch.int32, device=cuda)
    path = torch.tensor([[0, 2, -1, -1]], dtype=torch.int32, device=cuda)

    def run(cache, lens, w, par, pth, qs, **kw):
        out = F.mla_decode_tree(cache, qs[..., :128], qs[..., 128:], W_UK, W_UV, cos, sin, cfg, par, seq_lens=lens,
                                rotate_q=True, **kw)
        F.weigh_kv(w, cache, qs[..., :128], qs[..., 128:], W_UK, cos, sin, cfg, seq_lens=lens, rotate_q=True, **kw)
        weighed = w.clone()
        F.accept_kv(cache, lens, 4, pth, cfg, **kw)
        kept = F.evict_kv(cache, lens, w, cfg, 100, first=2, last=20, **kw)
        return out, weighed, kept

    small, n = near.clone()[None], torch.tensor([180], dtype=torch.int32, device=cuda)
    out0, w0, kept0 = run(small, n, torch.zeros(1, 192, device=cuda), parents, path, q)
    if paged:
        pool = kv.view(-1, 64, 576)[:LONG // 64]
        blocks = torch.tensor([[LONG // 64 - 1, LONG // 64 - 3, LONG // 64 - 2]], dtype=torch.int32, device=cuda)
        saved = pool[-3:].clone()
        for i, b in enumerate(blocks[0].tolist()):
            pool[b] = near[64 * i:64 * i + 64]
        lens = torch.tensor([180], dtype=torch.int32, device=cuda)
        out, w, kept = run(kv[0], lens, torch.zeros(1, 192, device=cuda), parents, path, q, block_table=blocks, block_size=64)
        rows = torch.cat([pool[b] for b in blocks[0].tolist()])
        pool[-3:] = saved
    else:
        cache = kv.view(REGIONS, LONG // REGIONS, 576)
        saved = cache[-1, :192].clone()
        cache[-1, :192] = near
        lens = torch.zeros(REGIONS, dtype=torch.int32, device=cuda)
        lens[-1] = 180
        w = torch.zeros(REGIONS, LONG // REGIONS, device=cuda)
        out, w, kept = run(cache, lens, w, parents.repeat(REGIONS, 1), path.repeat(REGIONS, 1), q.repeat(REGIONS, 1, 1))
        assert (out[:-4] == 0).all() and (w[:-1] == 0).all() and (kept[:-1] == -1).all()
        out, w, kept, rows, lens = out[-4:], w[-1:, :192], kept[-1:], cache[-1, :192].clone(), lens[-1:]
        cache[-1, :192] = saved
    assert_close(out.double().cpu().numpy(), out0.double().cpu().numpy(), "bf16")
    assert float((w - w0).norm() / w0.norm()) <= 1e-5 and (w[:, 180:] == 0).all()
    assert int(lens) == 100 and torch.equal(kept, kept0) and torch.equal(rows[:100], small[0, :100])
