"""Inputs and 64-bit references of the draft-tree and eviction tests, on the CPU.

Error bounds. The fp32 kernels (the plain forms, float32 caches) are held to
conftest's fp32 tolerances, the 16-bit matrix kernels to its 16-bit ones, as the
decode kernels whose roundings (queries, rope keys, probabilities) they share.

Weights (weigh_kv): scores are fp32 sums of K = kv_lora_rank + rope terms, of
operands that are exact or split so that 2^-16 of each is lost at most (two
bf16 parts of 8 significant bits each, and the product of the second ones), so
a score is off by at most e = (2^-16 + (K + 160) 2^-24) A, A = scale times the
sum of the terms' magnitudes (the absorbed query's own sum has 128 terms), a
weight by a factor within exp(+-2 e) (its exponent and its log-sum-exp), and an
exponential, its logarithm and the sum over n tokens, heads and partial sums by
(n heads + keys + 16) 2^-24 more, all of it relative to the weight.
Normwise: roundings of different terms are independent and at most 2^-18 of the
term (hi = x (1 + d), |d| <= 2^-9, of what is left 2^-9 again), so a score's
error has a standard deviation of at most 2^-18 B, B = scale times the root of
the sum of the squared terms, and its weight moves by at most twice that
(exponent and log-sum-exp): 2^-17 B of it. Scores of standard deviation 1 have B
of about 1, where 2^-17 and the fp32 sums stay below 1e-5; the tests hold
max(1e-5, 2^-17 B).
"""

from __future__ import annotations

import math
import random

import torch

from prompt_cases import as_double, rotate


def tree(n, seed, kind="random"):
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "star":
        return [-1] * n
    r = random.Random(seed)
    return [r.randint(max(-1, j - 7), j - 1) for j in range(n)]


def ancestors(parents):
    """Every node's set of itself and its ancestors."""
    sets = []
    for j, p in enumerate(parents):
        sets.append((sets[p] if 0 <= p < j else set()) | {j})
    return sets


def places(layout, s, n):
    """Rows of the flat cache that hold sequence s's first n positions."""
    kw = layout.kw
    if "block_table" in kw:
        b = kw["block_size"]
        t = kw["block_table"][s].cpu().long().clamp(0, layout.kv.shape[0] // b - 1)
        at = torch.arange(n)
        return t[at // b] * b + at % b
    if "seq_offsets" in kw:
        return torch.arange(n) + int(kw["seq_offsets"][s])
    return torch.arange(n) + s * layout.kv.shape[1]


def room(layout):
    """Shape of the row weights."""
    kw = layout.kw
    if "block_table" in kw:
        return tuple(kw["block_table"].shape[:1]) + (kw["block_table"].shape[1] * kw["block_size"],)
    return (layout.kv.shape[0],) if "seq_offsets" in kw else tuple(layout.kv.shape[:2])


def weight_places(layout, s, n):
    """Flat indexes of the weights of sequence s's first n positions."""
    shape = room(layout)
    return torch.arange(n) + (int(layout.kw["seq_offsets"][s]) if len(shape) == 1 else s * shape[1])


def scores(rows, q_nope, q_rope, W_UK, cos, sin, key_at, q_at, rotate_q):
    """(tokens, heads, rows) natural scores, the sums of their terms' magnitudes in latent space, and the roots of the
    sums of their squares."""
    heads, dn = q_nope.shape[1:]
    dc = W_UK.shape[1]
    scale = 1.0 / math.sqrt(dn + q_rope.shape[2])
    R = rotate(rows[:, dc:], cos[key_at], sin[key_at])
    qr = rotate(q_rope, cos[q_at][:, None], sin[q_at][:, None]) if rotate_q else q_rope
    W = W_UK.view(heads, dn, dc)
    qa = torch.einsum("thi,hic->thc", q_nope, W)
    x = scale * (torch.einsum("thc,kc->thk", qa, rows[:, :dc]) + torch.einsum("thr,kr->thk", qr, R))
    size = scale * (torch.einsum("thc,kc->thk", torch.einsum("thi,hic->thc", q_nope.abs(), W.abs()), rows[:, :dc].abs()) +
                    torch.einsum("thr,kr->thk", qr.abs(), rows[:, dc:].abs() * 2))
    root = scale * (torch.einsum("thc,kc->thk", qa ** 2, rows[:, :dc] ** 2) + torch.einsum("thr,kr->thk", qr ** 2, R ** 2)).sqrt()
    return x, size, root


def tree_reference(rows, q_nope, q_rope, W_UK, W_UV, cos, sin, parents, rotate_q):
    heads, dv, dc = q_nope.shape[1], W_UV.shape[0] // q_nope.shape[1], W_UV.shape[1]
    n = len(parents[0])
    out = torch.zeros(len(rows) * n, heads, dv, dtype=torch.float64)
    for s, r in enumerate(rows):
        L = r.shape[0]
        if L < n:
            continue
        sets = ancestors(parents[s])
        depth = torch.tensor([len(a) - 1 for a in sets])
        key_at = torch.cat([torch.arange(L - n), L - n + depth])
        t = slice(s * n, (s + 1) * n)
        x, _, _ = scores(r, q_nope[t], q_rope[t], W_UK, cos, sin, key_at, L - n + depth, rotate_q)
        sees = torch.zeros(n, L, dtype=torch.bool)
        sees[:, :L - n] = True
        for j, a in enumerate(sets):
            sees[j, [L - n + i for i in a]] = True
        # rows that a node does not see may hold anything
        x = torch.where(sees[:, None], x, torch.tensor(-math.inf, dtype=torch.float64))
        w = torch.softmax(x, -1)
        V = (r[:, :dc] @ W_UV.T).view(L, heads, dv)
        for j in range(n):
            out[s * n + j] = torch.einsum("hk,khd->hd", w[j][:, sees[j]], V[sees[j]])
    return out


def weigh_reference(rows, q_nope, q_rope, W_UK, cos, sin, n, rotate_q):
    """Of every sequence the weight that each row gets, the bound of its error, and the normwise one (the module's comment)."""
    outs, bounds, norms = [], [], []
    K = rows[0].shape[1] if rows else 0
    for s, r in enumerate(rows):
        L = r.shape[0]
        q_at = (torch.arange(n) + L - n).clamp(min=0)
        t = slice(s * n, (s + 1) * n)
        w, b, norm = torch.zeros(L, dtype=torch.float64), torch.zeros(L, dtype=torch.float64), 1e-5
        if L:
            x, size, root = scores(r, q_nope[t], q_rope[t], W_UK, cos, sin, torch.arange(L), q_at, rotate_q)
            for j in range(n):
                see = L - n + j + 1
                if see > 0:
                    p = torch.softmax(x[j, :, :see], -1)
                    off = (2.0 ** -16 + (K + 160) * 2.0 ** -24) * size[j, :, :see].amax(-1, keepdim=True)
                    w[:see] += p.sum(0)
                    norm = max(norm, 2.0 ** -17 * float(root[j, :, :see].max()))
                    b[:see] += (p * (torch.expm1(2 * off) + (n * q_nope.shape[1] + L + 16) * 2.0 ** -24)).sum(0)
        outs.append(w)
        bounds.append(b)
        norms.append(norm)
    return outs, bounds, norms


def evict_reference(w, keep, first, last):
    """Positions that stay of a sequence with the weights w (a list)."""
    L = len(w)
    if L <= keep:
        return list(range(L))
    key = [(-math.inf if math.isnan(x) else x) for x in w]
    nan = [math.isnan(x) for x in w]
    order = sorted(range(first, L - last), key=lambda i: (-key[i], nan[i], i))
    return sorted(list(range(first)) + order[:keep - first - last] + list(range(L - last, L)))


__all__ = ["tree", "ancestors", "places", "room", "weight_places", "tree_reference", "weigh_reference",
           "evict_reference", "as_double"]
