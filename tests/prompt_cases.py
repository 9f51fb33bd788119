"""Inputs and the 64-bit reference of the prompt and shared-prefix tests.

The reference is the definition, on the CPU in float64: K = c W_UK^T and V = c
W_UV^T per head, rope keys and (where asked) queries rotated by position, a
softmax over the keys that a token sees, the weighted sum of V. It also gives
what an error bound needs (below).

Error bound of the 16-bit forms, per output element. A rounding is off by at
most u = eps / 2 of the value (bf16 2^-8, fp16 2^-11). With w the softmax
weights, W = sum_k w_k |V_k| and A = max_k scale sum_i |q_i| |K_ki| (rope part
included):
  * V rounded, P rounded, the output rounded: u (W + W + |out|)
  * K and the rotated rope key rounded (and, where the queries are fp32 or are
    rotated on the way, q rounded): every score moves by at most r u A, r = 1 or
    2, so a weight moves by a factor within exp(+-2 r u A), and the output by at
    most (exp(2 r u A) - 1) W
plus fp32 sums, (512 + keys) 2^-24 of the same sums of magnitudes, which 1e-4 (W
+ A) covers up to 1000 keys. The absorbed form rounds q_abs and the rope key
and weights latent rows instead: there the sums of magnitudes run over the
latent dimension, where the framework's own 16-bit bound of the decode kernels
(conftest.assert_close) applies. Roundings are independent, so the normwise
error is far below the bound: conftest's 1e-2 holds for every form.
"""

from __future__ import annotations

import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def tables(rows: int, d_r: int = 64):
    freq = 10000.0 ** (-torch.arange(0, d_r, 2, dtype=torch.float64) / d_r)
    angle = torch.arange(max(rows, 1), dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def rotate(x, cos, sin):
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def reference(rows, q_nope, q_rope, W_UK, W_UV, cos, sin, new, prefix=None, rotate_q=False):
    """rows: per sequence (L, dc + dR); q (tokens, H, .); new: tokens per sequence; everything float64 on the CPU.
    Returns out, W, A: (tokens, H, dv), (tokens, H, dv), (tokens, H)."""
    heads, dn = q_nope.shape[1:]
    dv, dc = W_UV.shape[0] // heads, W_UV.shape[1]
    d_r = q_rope.shape[2]
    scale = 1.0 / math.sqrt(dn + d_r)
    out = torch.zeros(q_nope.shape[0], heads, dv, dtype=torch.float64)
    mass, size = torch.zeros_like(out), torch.zeros(q_nope.shape[0], heads, dtype=torch.float64)
    t = 0
    for s, (r, n) in enumerate(zip(rows, new)):
        L = r.shape[0]
        K = (r[:, :dc] @ W_UK.T).view(L, heads, dn)
        V = (r[:, :dc] @ W_UV.T).view(L, heads, dv)
        R = rotate(r[:, dc:], cos[:L], sin[:L])
        for j in range(n):
            p = L - n + j
            see = max(p + 1, min(prefix[s], L) if prefix is not None else 0, 0)
            if see:
                qr = rotate(q_rope[t], cos[max(p, 0)], sin[max(p, 0)]) if rotate_q else q_rope[t]
                x = scale * (torch.einsum("hi,khi->hk", q_nope[t], K[:see]) + qr @ R[:see].T)
                w = torch.softmax(x, -1)
                out[t] = torch.einsum("hk,khd->hd", w, V[:see])
                mass[t] = torch.einsum("hk,khd->hd", w, V[:see].abs())
                size[t] = scale * (torch.einsum("hi,khi->hk", q_nope[t].abs(), K[:see].abs()) + qr.abs() @ R[:see].abs().T).amax(-1)
            t += 1
    return out, mass, size


def check(got, ref, u, roundings, out_u, what=""):
    """Asserts the bound of the module's comment, and the normwise one."""
    out, mass, size = ref
    got = got.double().cpu()
    assert got.shape == out.shape
    assert torch.isfinite(got).all(), f"{what}: non-finite output"
    bound = 2 * u * mass + torch.expm1(2 * roundings * u * size)[..., None] * mass + out_u * out.abs() + 1e-4 * (
        mass + size[..., None])
    over = (got - out).abs() - bound
    assert (over <= 0).all(), f"{what}: {over.max():.3e} over the bound at {over.argmax()}"
    if out.norm() > 0:
        assert (got - out).norm() <= 1e-2 * out.norm(), f"{what}: normwise {(got - out).norm() / out.norm():.3e}"


def weights(heads, dtype, seed, dc=512, dn=128, dv=128):
    g = torch.Generator().manual_seed(seed)
    return ((torch.randn(heads * dn, dc, generator=g) / dc ** 0.5).to(dtype),
            (torch.randn(heads * dv, dc, generator=g) / dc ** 0.5).to(dtype))


def as_double(t):
    return t.detach().cpu().to(torch.float32).double()


class Layout:
    """The same sequences' rows in one of the cache layouts; rows outside the sequences hold `junk`."""

    def __init__(self, kind, rows, dtype, device, junk=float("nan"), block=64, seed=0):
        self.kw = {}
        width = rows[0].shape[1]
        lens = [r.shape[0] for r in rows]
        if dtype == torch.float8_e4m3fn and not math.isnan(junk):
            junk = float("nan")
        if kind == "uniform":
            assert len(set(lens)) == 1
            self.kv = torch.stack(rows)
        elif kind == "capacity":
            cap = -(-(max(lens) + 1) // 32) * 32
            self.kv = torch.full((len(rows), cap, width), junk)
            for s, r in enumerate(rows):
                self.kv[s, :lens[s]] = r
            self.kw["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=device)
        elif kind == "packed":
            self.kv = torch.cat(rows) if sum(lens) else torch.zeros(0, width)
            at = [0]
            for n in lens:
                at.append(at[-1] + n)
            self.kw["seq_offsets"] = torch.tensor(at, dtype=torch.int32, device=device)
        elif kind == "packed_capacity":  # regions of their own sizes, filled in part
            at, parts = [0], []
            for s, r in enumerate(rows):
                spare = (7 * s) % 50
                parts += [r, torch.full((spare, width), junk)]
                at.append(at[-1] + lens[s] + spare)
            self.kv = torch.cat(parts)
            self.kw["seq_offsets"] = torch.tensor(at, dtype=torch.int32, device=device)
            self.kw["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=device)
        else:
            g = torch.Generator().manual_seed(seed)
            per = max(-(-max(lens) // block), 1) + 1
            order = torch.randperm(len(rows) * per + 2, generator=g)
            pool = torch.full((order.numel() * block, width), junk)
            table = torch.full((len(rows), per), 10 ** 6, dtype=torch.int32)
            for s, r in enumerate(rows):
                for i in range(-(-lens[s] // block)):
                    b = int(order[s * per + i])
                    table[s, i] = b
                    part = r[i * block:(i + 1) * block]
                    pool[b * block:b * block + part.shape[0]] = part
            self.kv = pool
            self.kw = {"block_table": table.to(device), "block_size": block,
                       "seq_lens": torch.tensor(lens, dtype=torch.int32, device=device)}
        self.kv = self.kv.to(dtype).to(device).contiguous()
