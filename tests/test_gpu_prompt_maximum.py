"""The running maximum of the prompt kernels: scores that rise, fall and jump by tens from one tile of 64 keys to the
next, so that sums and outputs are rescaled, once per tile or once in several, by powers between 2^-8 and 2^-100.

Keys are constant within a tile (one latent column holds the tile's level, and W_UK reads nothing else) and values do not
depend on the level (W_UV does not read that column), so the weights are known to a few roundings however large the
scores: the bound of tests/prompt_cases.py with A, the largest score, at most 72. Tokens of one wave have scores of
different slopes. That the bound tells a rescale that is missing is tested on the CPU, in an oracle that leaves it out."""

from __future__ import annotations

import math

import pytest
import torch

from prompt_cases import U, as_double, check, reference, rotate, tables

from latent_attn import MLAConfig
from latent_attn import functional as F

EXPANDED = 2
HEADS = 3
SLOPES = (3.0, 6.0, 12.0)  # of a token's scores per level, in powers of e
LEVELS = {"up": [0, 1, 2, 3, 4, 5, 6], "jumps": [2, 0, 3, 1, 6, 5, 6], "one step": [0, 0, 0, 0, 6, 6, 6],
          "down": [6, 5, 4, 3, 2, 1, 0]}


def inputs(levels, tokens, dtype, per=64):
    g = torch.Generator().manual_seed(len(levels) + tokens)
    rows = torch.randn(per * len(levels) - 7, 576, generator=g)  # the last tile is cut
    rows[:, 0] = torch.tensor(levels, dtype=torch.float32).repeat_interleave(per)[:rows.shape[0]]
    rows[:, 512:] = 0
    sign = torch.randint(0, 2, (HEADS, 128), generator=g) * 2.0 - 1.0
    W_UK = torch.zeros(HEADS * 128, 512)
    W_UK[:, 0] = sign.flatten()
    W_UV = torch.randn(HEADS * 128, 512, generator=g) / 512 ** 0.5
    W_UV[:, 0] = 0
    slope = torch.tensor(SLOPES).repeat(tokens * HEADS)[:tokens * HEADS].view(tokens, HEADS)
    q = torch.randn(tokens, HEADS, 192, generator=g)
    q[..., :128] = slope[..., None] * math.sqrt(192) / 128 * sign
    return rows.to(dtype), q.to(dtype), W_UK.to(dtype), W_UV.to(dtype)


def expected(rows, q, W_UK, W_UV, new, cos, sin):
    return reference([as_double(rows)], as_double(q[..., :128]), as_double(q[..., 128:]), as_double(W_UK), as_double(W_UV),
                     as_double(cos), as_double(sin), [new])


def limit(ref, u, roundings, out_u):
    """The bound of tests/prompt_cases.py per element."""
    out, mass, size = ref
    return 2 * u * mass + torch.expm1(2 * roundings * u * size)[..., None] * mass + out_u * out.abs() + 1e-4 * (
        mass + size[..., None])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("levels", LEVELS)
@pytest.mark.parametrize("tokens", [441, 5])
def test_prompts(cuda, levels, tokens, dtype):
    rows, q, W_UK, W_UV = inputs(LEVELS[levels], tokens, dtype)
    cos, sin = tables(rows.shape[0])
    ref = expected(rows, q, W_UK, W_UV, tokens, cos, sin)
    dev = [t.to(cuda) for t in (rows[None], q[..., :128], q[..., 128:], W_UK, W_UV, cos, sin)]
    got = F.mla_prefill(*dev, MLAConfig(5120, 512, 128, 64, HEADS, 128), kernel_variant=EXPANDED)
    check(got, ref, U[dtype], 1, U[dtype], f"{levels} {dtype}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("levels", LEVELS)
def test_key_parts(cuda, levels, dtype):
    """Few tokens over four tiles of every level: parts of the keys, joined, whose maxima lie far apart."""
    rows, q, W_UK, W_UV = inputs(LEVELS[levels], 3, dtype, per=256)
    cos, sin = tables(rows.shape[0])
    ref = expected(rows, q, W_UK, W_UV, 3, cos, sin)
    dev = [t.to(cuda) for t in (rows[None], q[..., :128], q[..., 128:], W_UK, W_UV, cos, sin)]
    got = F.mla_prefill(*dev, MLAConfig(5120, 512, 128, 64, HEADS, 128), kernel_variant=EXPANDED)
    check(got, ref, U[dtype], 1, U[dtype], f"parts {levels} {dtype}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("levels", LEVELS)
@pytest.mark.parametrize("cut", [150, 320])
def test_shared_steps(cuda, levels, cut, dtype):
    """The first rows as an expanded prefix, the others every sequence's own; queries are scaled and rounded on the way
    (two roundings per score). The own rows' step of 3 heads is in float32.

    Per element only: the normwise bound of prompt_cases counts on roundings that are independent, and these are not.
    All 128 dims of a query have one magnitude and so one rounding error, which moves every score over the prefix by the
    same factor 1 + d, |d| <= u, and no own score. Where both parts hold keys of level 6, the weights of the two move
    against each other by e^(d s), s = 72: by up to a third in bf16."""
    rows, q, W_UK, W_UV = inputs(LEVELS[levels], 9, dtype)
    cos, sin = tables(rows.shape[0])
    q = q.float()
    parts = [expected(rows, q[i:i + 1], W_UK, W_UV, 1, cos, sin) for i in range(9)]
    ref = [torch.cat([p[k] for p in parts]) for k in range(3)]
    cfg = MLAConfig(5120, 512, 128, 64, HEADS, 128)
    W_UK, W_UV, cos, sin, rows, q = (t.to(cuda) for t in (W_UK, W_UV, cos, sin, rows, q))
    prefix = F.expand_prefix(rows[:cut].contiguous(), W_UK, W_UV, cos, sin, cfg)
    own = rows[cut:].expand(9, -1, -1).contiguous()
    got = F.mla_decode_shared(prefix, own, q[..., :128].contiguous(), q[..., 128:].contiguous(), W_UK, W_UV, cos, sin, cfg,
                              kernel_variant=EXPANDED)
    over = (got.double().cpu() - ref[0]).abs() - limit(ref, U[dtype], 2, 0.0)
    assert (over <= 0).all(), f"shared {levels} {dtype}: {over.max():.3e} over the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [2, 8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_parts_equal_one_part(cuda, heads, dtype):
    """A sequence alone runs in parts of its keys; among 600 others (which have one key each) in one part. Expanded keys,
    values and scores are the same numbers in both. Different are the exponentials' roundings to 16 bits (another maximum
    before them: u of sum w |V| each), the order of fp32 sums and, where the output is rounded, that rounding."""
    L, n, others = 2000, 3, 600
    cfg = MLAConfig(5120, 512, 128, 64, heads, 128)
    g = torch.Generator().manual_seed(heads)
    rows = torch.randn(L, 576, generator=g).to(dtype)
    W_UK, W_UV = ((torch.randn(heads * 128, 512, generator=g) / 22).to(dtype) for _ in range(2))
    cos, sin = tables(L)
    q = torch.randn(n, heads, 192, generator=g).to(dtype)
    mass = expected(rows, torch.cat([q[..., :128], rotated(q[..., 128:], cos, sin, L - n)], -1), W_UK, W_UV, n, cos, sin)[1]
    W_UK, W_UV, cos, sin, rows, q = (t.to(cuda) for t in (W_UK, W_UV, cos, sin, rows, q))

    def run(kv, queries, k_at, q_at):
        return F.mla_prefill(kv, queries[..., :128], queries[..., 128:], W_UK, W_UV, cos, sin, cfg, rotate_q=True,
                             q_offsets=torch.tensor(q_at, dtype=torch.int32, device=cuda), out_dtype=torch.float32,
                             seq_offsets=torch.tensor(k_at, dtype=torch.int32, device=cuda), kernel_variant=EXPANDED)

    alone = run(rows, q, [0, L], [0, n])
    many = run(torch.cat([rows, rows[:others]]), torch.cat([q, q[:1].expand(others, -1, -1)]),
               [0, *range(L, L + others + 1)], [0, *range(n, n + others + 1)])[:n]
    assert ((alone - many).abs().double().cpu() <= (2 * U[dtype] + 1e-4) * mass).all()


def rotated(x, cos, sin, first):
    at = torch.arange(first, first + x.shape[0])
    return rotate(as_double(x), as_double(cos)[at][:, None], as_double(sin)[at][:, None])


@pytest.mark.parametrize("roundings", [1, 2])
@pytest.mark.parametrize("mistake", ["sum", "output", "start"])
def test_the_bound_sees_a_missing_rescale(mistake, roundings):
    """The kernel's loop over tiles, in float64: with each part of its rescale left out some token passes the bound, with all
    of them none comes near it."""
    for dtype in (torch.float16, torch.bfloat16):
        worst = {False: 0.0, True: 0.0}
        for levels in LEVELS.values():
            rows, q, W_UK, W_UV = inputs(levels, 6, dtype)
            cos, sin = tables(rows.shape[0])
            ref = expected(rows, q, W_UK, W_UV, 6, cos, sin)
            bound = limit(ref, U[dtype], roundings, U[dtype])
            c = as_double(rows)[:, :512]
            K, V = ((c @ as_double(W).T).view(-1, HEADS, 128) for W in (W_UK, W_UV))
            for t in range(6):
                see = rows.shape[0] - 6 + t + 1
                for h in range(HEADS):
                    s = (K[:see, h] @ as_double(q)[t, h, :128]) / math.sqrt(192) * math.log2(math.e)
                    for wrong in (False, True):
                        m = used = total = 0.0
                        o = torch.zeros(128, dtype=torch.float64)
                        for at in range(0, see, 64):
                            x = s[at:at + 64] - used
                            top = x.max().item()
                            if at == 0 or top > 8:
                                f = 0.0 if at == 0 else 2.0 ** -top
                                m += top
                                x = x - top
                                if not (wrong and mistake == "sum"):
                                    total *= f
                                if not (wrong and mistake == "output"):
                                    o *= f
                                if at == 0 or not (wrong and mistake == "start"):
                                    used = m
                            p = torch.exp2(x.clamp(max=900))
                            total += p.sum().item()
                            o += p @ V[at:at + 64, h][:p.shape[0]]
                        worst[wrong] = max(worst[wrong], ((o / total - ref[0][t, h]).abs() / bound[t, h]).max().item())
        assert worst[False] < 1e-3 and worst[True] > 1, worst
