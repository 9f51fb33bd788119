"""The form that an automatic mla_prefill or mla_decode_shared call takes. A call's workspace size tells its form: each
carves other pieces. (Sizes are counted on the host, from the descriptor alone, on the device that would run the call.)"""

from __future__ import annotations

import ctypes

import pytest
import torch

from conftest import assert_close
from prompt_cases import Layout, as_double, reference, tables, weights

from latent_attn import MLAConfig, capi
from latent_attn import functional as F

pytestmark = pytest.mark.gpu

EXPANDED, ABSORBED = 2, 3
LATENT, OF_EXPANDED = 1, 2
AT = 1 << 20  # an aligned address that sizes are counted with and nothing reads


def config(heads):
    return MLAConfig(5120, 512, 128, 64, heads, 128)


def prefill_size(form, heads, batch, new, rows, block=0, kv=AT, dtype=capi.LA_DTYPE_BF16):
    a = capi.PrefillArgs(kv_dtype=dtype, num_seqs=batch, tokens=batch * new, q_dtype=capi.LA_DTYPE_BF16, rotate_q=1,
                         w_uk_dtype=capi.LA_DTYPE_BF16, w_uv_dtype=capi.LA_DTYPE_BF16, out_dtype=capi.LA_DTYPE_BF16,
                         rope_rows=rows, cfg=capi.config(config(heads)), kernel_variant=form)
    for f in ("q_nope", "q_rope", "W_UK", "W_UV", "rope_cos", "rope_sin", "output"):
        setattr(a, f, AT)
    a.kv_cache = kv
    if block:
        per = -(-rows // block)
        a.block_table = a.seq_lens = AT
        a.block_size, a.blocks_per_seq, a.total_rows = block, per, batch * per * block
    else:
        a.seq_len, a.total_rows = rows, batch * rows
    return capi.load().la_mla_prefill_workspace_size(ctypes.byref(a))


@pytest.mark.parametrize("case", [
    dict(heads=128, batch=16, new=4, rows=2000, block=16),
    dict(heads=128, batch=16, new=4, rows=2000, block=16, dtype=capi.LA_DTYPE_FP8_E4M3),
    dict(heads=128, batch=1, new=128, rows=8192, block=16),
    dict(heads=16, batch=16, new=4, rows=2000, block=48),
    dict(heads=128, batch=1, new=4, rows=2000, block=1),
    dict(heads=128, batch=4, new=16, rows=1000),
    dict(heads=128, batch=1, new=1, rows=8200),
    dict(heads=8, batch=16, new=4, rows=2000, block=64),
    dict(heads=8, batch=1, new=64, rows=8192),
    dict(heads=17, batch=1, new=8, rows=4000, block=64),
    dict(heads=1, batch=16, new=4, rows=2000, block=64),
    dict(heads=128, batch=16, new=4, rows=2048, block=64, kv=AT + 2),
])
def test_no_valu_step_beside_the_expanded_form(cuda, case):
    """Pages, regions, heads and addresses without a matrix kernel for the absorbed form's step."""
    auto, expanded, absorbed = (prefill_size(form, **case) for form in (0, EXPANDED, ABSORBED))
    assert expanded != absorbed and absorbed > 0
    assert auto == expanded


@pytest.mark.parametrize("case", [
    dict(heads=128, batch=16, new=4, rows=2000, block=64),
    dict(heads=128, batch=16, new=4, rows=2000, block=32),
    dict(heads=128, batch=1, new=4, rows=1024),
    dict(heads=128, batch=1, new=4, rows=1024 + 32),
    dict(heads=16, batch=16, new=4, rows=4096, block=128),
    dict(heads=48, batch=16, new=2, rows=4096, block=64),
    dict(heads=1, batch=1, new=1, rows=131072, block=64),  # on the VALU, which beats the expansion for one head
])
def test_a_few_tokens_stay_absorbed(cuda, case):
    auto, expanded, absorbed = (prefill_size(form, **case) for form in (0, EXPANDED, ABSORBED))
    assert expanded != absorbed and absorbed > 0
    assert auto == absorbed


def shared_size(form, heads, batch, prefix, at=AT):
    a = capi.SharedArgs(prefix=at, prefix_len=prefix, expanded=AT, output=AT, out_dtype=capi.LA_DTYPE_BF16,
                        kernel_variant=form)
    a.own = capi.DecodeArgs(kv_dtype=capi.LA_DTYPE_BF16, num_seqs=batch, seq_len=64, total_rows=64 * batch,
                            queries_per_seq=1, w_uk_dtype=capi.LA_DTYPE_BF16, w_uv_dtype=capi.LA_DTYPE_BF16,
                            rope_rows=prefix + 64, cfg=capi.config(config(heads)))
    for f in ("kv_cache", "q_nope", "q_rope", "W_UK", "W_UV", "rope_cos", "rope_sin"):
        setattr(a.own, f, AT)
    return capi.load().la_mla_decode_shared_workspace_size(ctypes.byref(a))


@pytest.mark.parametrize("case", [
    dict(heads=8, batch=1, prefix=64), dict(heads=8, batch=1, prefix=32768), dict(heads=17, batch=2, prefix=4000),
    dict(heads=17, batch=8, prefix=32768), dict(heads=1, batch=8, prefix=32768), dict(heads=24, batch=1, prefix=32768),
    dict(heads=128, batch=1, prefix=8192, at=AT + 2),
])
def test_no_valu_step_over_an_expanded_prefix(cuda, case):
    auto, latent, expanded = (shared_size(form, **case) for form in (0, LATENT, OF_EXPANDED))
    assert latent != expanded and latent > 0
    assert auto == expanded


@pytest.mark.parametrize("case", [dict(heads=128, batch=1, prefix=8192), dict(heads=8, batch=8, prefix=32768),
                                  dict(heads=16, batch=1, prefix=8192)])
def test_a_few_queries_read_the_latent_rows(cuda, case):
    auto, latent, expanded = (shared_size(form, **case) for form in (0, LATENT, OF_EXPANDED))
    assert latent != expanded and latent > 0
    assert auto == latent


@pytest.mark.parametrize("heads,rows,new,block", [(16, [300, 90], [3, 1], 16), (128, [200, 33], [2, 4], 48),
                                                  (8, [700, 1], [4, 1], 64), (17, [260, 64], [4, 4], 64)])
def test_automatic_calls(cuda, heads, rows, new, block):
    """Such calls themselves: the expanded form's bits, and right."""
    g = torch.Generator().manual_seed(heads)
    data = [torch.randn(n, 576, generator=g).bfloat16().float() for n in rows]
    layout = Layout("paged", data, torch.bfloat16, cuda, block=block)
    q = torch.randn(sum(new), heads, 192, generator=g).bfloat16().to(cuda)
    W_UK, W_UV = (w.to(cuda) for w in weights(heads, torch.bfloat16, 2))
    cos, sin = (t.to(cuda) for t in tables(max(rows)))
    off = torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device=cuda)
    run = lambda form: F.mla_prefill(layout.kv, q[..., :128], q[..., 128:], W_UK, W_UV, cos, sin, config(heads),
                                     q_offsets=off, rotate_q=True, kernel_variant=form, **layout.kw)
    got = run(0)
    assert torch.equal(got, run(EXPANDED))
    ref = reference([d.double() for d in data], as_double(q[..., :128]), as_double(q[..., 128:]), as_double(W_UK),
                    as_double(W_UV), as_double(cos), as_double(sin), new, None, True)
    assert_close(got.double().cpu().numpy(), ref[0].numpy(), "bf16", f"{heads} heads, pages of {block}")


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


def small_reference(rows, q, W_UK, W_UV, heads, dn, dv):
    """One sequence's causal attention from the definition, float64, without rotation; q (n, heads, dn + dR), the last n
    rows' queries."""
    dc = W_UK.shape[1]
    c, r = rows[:, :dc].double(), rows[:, dc:].double()
    K = (c @ W_UK.double().T).view(-1, heads, dn)
    V = (c @ W_UV.double().T).view(-1, heads, dv)
    q = q.double()
    x = torch.matmul(q[..., :dn].transpose(0, 1), K.permute(1, 2, 0).contiguous())
    x = x + torch.matmul(q[..., dn:].transpose(0, 1), r.T.contiguous())
    x /= (q.shape[2]) ** 0.5
    n, L = q.shape[0], rows.shape[0]
    x = x.masked_fill(torch.arange(L, device=x.device) > torch.arange(L - n, L, device=x.device)[:, None], -float("inf"))
    return torch.matmul(torch.softmax(x, -1), V.transpose(0, 1).contiguous()).transpose(0, 1)


def unrotated(rows, d_r, device):
    return torch.ones(rows, d_r // 2, device=device), torch.zeros(rows, d_r // 2, device=device)


# float32 throughout. A score sums at most dc + dn + dR = 88 rounded products, whose magnitudes here add up to less than
# 60 (after the scale), so it is off by at most 88 x 2^-24 x 60 = 3.2e-4, a weight by a factor within 1 +- 6.4e-4, and an
# output by that of sum w |V| < 6: 3.9e-3. (V's own sums of 64 products add 64 x 2^-24 x 10 = 4e-5.)
CLOSE = 4e-3


@pytest.mark.parametrize("heads,tokens,dims,doc", [
    (128, 1 << 17, (16, 8, 8, 8), 64),     # 2^24 workgroups of 256 threads: one more than a grid holds
    (1, (1 << 20) + 640, (16, 8, 8, 8), 64),  # absorption in blocks of 16 tokens: more than 65,535 of them
    (1, (1 << 20) + 640, (64, 16, 8, 8), 64),  # ... on the matrix cores
])
def test_plain_calls_past_one_grid(cuda, heads, tokens, dims, doc):
    dc, dn, d_r, dv = dims
    cfg = MLAConfig(64, dc, dn, d_r, heads, dv)
    g = torch.Generator(device=cuda).manual_seed(1)
    kv = torch.randn(tokens, dc + d_r, generator=g, device=cuda)
    W_UK, W_UV = (torch.randn(heads * d, dc, generator=g, device=cuda) / dc ** 0.5 for d in (dn, dv))
    q = torch.randn(tokens, heads, dn + d_r, generator=g, device=cuda)
    off = torch.arange(0, tokens + 1, doc, device=cuda).int()
    cos, sin = unrotated(doc, d_r, cuda)
    got = F.mla_prefill(kv, q[..., :dn], q[..., dn:], W_UK, W_UV, cos, sin, cfg, q_offsets=off, seq_offsets=off,
                        kernel_variant=1)
    for at in (0, tokens // doc // 2 * doc, tokens - doc):
        ref = small_reference(kv[at:at + doc], q[at:at + doc], W_UK, W_UV, heads, dn, dv)
        assert (got[at:at + doc].double() - ref).abs().max() <= CLOSE, at


def test_an_absorbed_call_past_one_grid(cuda):
    """600,000 tokens' projections in blocks of 8: more than 65,535 of them."""
    B, n, cap, (dc, dn, d_r, dv) = 10000, 60, 64, (16, 8, 8, 8)
    cfg = MLAConfig(64, dc, dn, d_r, 1, dv)
    g = torch.Generator(device=cuda).manual_seed(2)
    kv = torch.randn(B, cap, dc + d_r, generator=g, device=cuda)
    W_UK, W_UV = (torch.randn(d, dc, generator=g, device=cuda) / dc ** 0.5 for d in (dn, dv))
    q = torch.randn(B * n, 1, dn + d_r, generator=g, device=cuda)
    cos, sin = unrotated(cap, d_r, cuda)
    got = F.mla_prefill(kv, q[..., :dn], q[..., dn:], W_UK, W_UV, cos, sin, cfg, kernel_variant=ABSORBED)
    for b in (0, 8737, 8738, B - 1):
        ref = small_reference(kv[b], q[b * n:(b + 1) * n], W_UK, W_UV, 1, dn, dv)
        assert (got[b * n:(b + 1) * n].double() - ref).abs().max() <= CLOSE, b


def test_a_shared_step_past_one_grid(cuda):
    """The prefix's step has batch x heads query heads: 76,800 where a grid's y holds 65,535."""
    B, heads, P, own, (dc, dn, d_r, dv) = 600, 128, 70, 5, (16, 8, 8, 8)
    cfg = MLAConfig(64, dc, dn, d_r, heads, dv)
    g = torch.Generator(device=cuda).manual_seed(3)
    front, kv = torch.randn(P, dc + d_r, generator=g, device=cuda), torch.randn(B, own, dc + d_r, generator=g, device=cuda)
    W_UK, W_UV = (torch.randn(heads * d, dc, generator=g, device=cuda) / dc ** 0.5 for d in (dn, dv))
    q_nope, q_rope = (torch.randn(B, heads, d, generator=g, device=cuda) for d in (dn, d_r))
    cos, sin = unrotated(P + own, d_r, cuda)
    got = F.mla_decode_shared(front, kv, q_nope, q_rope, W_UK, W_UV, cos, sin, cfg)
    for b in (0, 511, 512, B - 1):
        ref = small_reference(torch.cat([front, kv[b]]), torch.cat([q_nope, q_rope], -1)[b:b + 1], W_UK, W_UV, heads, dn, dv)
        assert (got[b:b + 1].double() - ref).abs().max() <= CLOSE, b


@pytest.mark.parametrize("heads", [16, 3])
@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float32])
def test_a_prefix_and_no_room_for_own_rows(cuda, heads, kv):
    """Own caches of no rows at all: the prefix alone."""
    g = torch.Generator().manual_seed(5)
    front = torch.randn(90, 576, generator=g).to(kv).to(cuda)
    W_UK, W_UV = (w.to(cuda) for w in weights(heads, kv, 6))
    cos, sin = (t.to(cuda) for t in tables(90))
    q_nope, q_rope = (torch.randn(2, heads, d, generator=g).to(cuda) for d in (128, 64))
    args = (torch.zeros(2, 0, 576, dtype=kv, device=cuda), q_nope, q_rope, W_UK, W_UV, cos, sin, config(heads))
    ref = reference([as_double(front)] * 2, as_double(q_nope), as_double(q_rope), as_double(W_UK), as_double(W_UV),
                    as_double(cos), as_double(sin), [1, 1])[0]
    got = [F.mla_decode_shared(front, *args)]
    if kv == torch.bfloat16:
        prefix = F.expand_prefix(front, W_UK, W_UV, cos, sin, config(heads))
        got += [F.mla_decode_shared(prefix, *args, kernel_variant=form) for form in (LATENT, OF_EXPANDED)]
    for x in got:
        assert_close(x.double().cpu().numpy(), ref.numpy(), "bf16" if kv == torch.bfloat16 else "f32", f"{heads} {kv}")
