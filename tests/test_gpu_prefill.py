"""GPU parity of functional.mla_prefill (la_mla_prefill) against the 64-bit
reference of tests/prompt_cases.py: every form, cache layout, cache and query
type, odd and empty lengths, masks, strides, and its use in a run of the
framework's calls and in a captured graph."""

from __future__ import annotations

import pytest
import torch

from conftest import assert_close
from prompt_cases import U, Layout, as_double, check, reference, tables, weights

from latent_attn import MLAConfig
from latent_attn import functional as F

pytestmark = pytest.mark.gpu

AUTO, PLAIN, EXPANDED, ABSORBED = 0, 1, 2, 3


def config(heads, dc=512, dn=128, d_r=64, dv=128):
    return MLAConfig(5120, dc, dn, d_r, heads, dv)


class Case:
    def __init__(self, cuda, layout, rows, new, heads=4, kv=torch.bfloat16, q=torch.bfloat16, w=None, prefix=None,
                 rotate_q=True, block=64, seed=1, dims=(512, 128, 64, 128), pad=0, scale=1.0):
        dc, dn, d_r, dv = dims
        self.cfg, self.kv_type, self.q_type = config(heads, dc, dn, d_r, dv), kv, q
        g = torch.Generator().manual_seed(seed)
        data = [(torch.randn(n, dc + d_r, generator=g) * scale).to(kv).float() for n in rows]
        self.layout = Layout(layout, data, kv, cuda, block=block, seed=seed)
        self.rows = [d.double() for d in data]
        tokens = sum(new) + pad
        self.q = torch.randn(tokens, heads, dn + d_r, generator=g).to(q).to(cuda)
        w = w or (kv if kv in U else torch.bfloat16 if kv != torch.float32 else torch.float32)
        self.W_UK, self.W_UV = (x.to(cuda) for x in weights(heads, w, seed + 1, dc, dn, dv))
        cos, sin = tables(max(rows), d_r)
        self.cos, self.sin = cos.to(cuda), sin.to(cuda)
        self.new, self.prefix, self.rotate_q, self.dn = new, prefix, rotate_q, dn
        at = [0]
        for n in new:
            at.append(at[-1] + n)
        self.kw = dict(self.layout.kw)
        self.kw["q_offsets"] = torch.tensor(at, dtype=torch.int32, device=cuda)
        if prefix is not None:
            self.kw["prefix_lens"] = torch.tensor(prefix, dtype=torch.int32, device=cuda)

    def run(self, **kw):
        kw = {**self.kw, "rotate_q": self.rotate_q, **kw}
        return F.mla_prefill(self.layout.kv, self.q[..., :self.dn], self.q[..., self.dn:], self.W_UK, self.W_UV,
                             self.cos, self.sin, self.cfg, **kw)

    def reference(self):
        q = as_double(self.q)
        return reference(self.rows, q[..., :self.dn], q[..., self.dn:], as_double(self.W_UK), as_double(self.W_UV),
                         as_double(self.cos), as_double(self.sin), self.new, self.prefix, self.rotate_q)

    def check(self, got, form, what=""):
        ref = self.reference()
        if self.kv_type == torch.float32:
            assert got.dtype == self.q_type
            if got.dtype == torch.float32:
                assert_close(got.cpu().numpy(), ref[0].numpy(), "f32", what)
            else:  # fp32 sums, one rounding of the output
                bound = U[got.dtype] * ref[0].abs() + 1e-4
                assert ((got.double().cpu() - ref[0]).abs() <= bound).all(), what
            return
        u = U[torch.float16 if self.kv_type == torch.float16 else torch.bfloat16]
        if form == EXPANDED:
            q_rounds = self.rotate_q or self.q_type != (torch.float16 if self.kv_type == torch.float16 else torch.bfloat16)
            check(got, ref, u, 2 if q_rounds else 1, U.get(got.dtype, 0.0), what)
        else:
            assert_close(got.double().cpu().numpy(), ref[0].numpy(), "bf16", what)


ODD_ROWS, ODD_NEW = [1, 63, 64, 65, 200, 130], [1, 5, 64, 65, 130, 129]


@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("layout", ["packed", "capacity", "packed_capacity", "paged"])
def test_expanded_layouts(cuda, layout, kv):
    c = Case(cuda, layout, ODD_ROWS, ODD_NEW, kv=kv, q=torch.float16 if kv == torch.float16 else torch.bfloat16)
    c.check(c.run(kernel_variant=EXPANDED), EXPANDED, f"{layout} {kv}")


@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.float32])
@pytest.mark.parametrize("layout,form", [("capacity", ABSORBED), ("paged", ABSORBED), ("packed", PLAIN),
                                         ("capacity", PLAIN), ("paged", PLAIN), ("packed_capacity", PLAIN)])
def test_other_forms(cuda, layout, form, kv):
    c = Case(cuda, layout, ODD_ROWS, [1, 5, 8, 3, 1, 7], heads=16, kv=kv, q=torch.float32)
    c.check(c.run(kernel_variant=form), form, f"{layout} {kv}")


@pytest.mark.parametrize("form", [PLAIN, EXPANDED, ABSORBED])
def test_empty_rows_and_more_tokens_than_rows(cuda, form):
    """A sequence without rows, one with more new tokens than rows (its first tokens see nothing), one without new
    tokens, and padding behind the last sequence: zeros there, the rest as ever."""
    c = Case(cuda, "capacity", [0, 3, 70, 40], [2, 9, 0, 40], heads=16, pad=5)
    got = c.run(kernel_variant=form)
    c.check(got, form, "empty")
    assert (got[:2] == 0).all() and (got[2:8] == 0).all() and (got[-5:] == 0).all()
    assert (got[8] != 0).any()


@pytest.mark.parametrize("form", [PLAIN, EXPANDED, ABSORBED])
@pytest.mark.parametrize("prefix", [[0, 7, 64, 500, 1], [1000] * 5])
def test_prefix_mask(cuda, form, prefix):
    c = Case(cuda, "capacity", [50, 64, 130, 129, 1], [50, 60, 100, 3, 1], heads=16, prefix=prefix)
    c.check(c.run(kernel_variant=form), form, "prefix")


@pytest.mark.parametrize("heads", [1, 3, 8, 16, 17])
@pytest.mark.parametrize("n,L", [(1, 1), (1, 300), (33, 33), (127, 500), (257, 257)])
def test_heads_and_lengths(cuda, heads, n, L):
    c = Case(cuda, "uniform", [L, L], [n, n], heads=heads)
    c.check(c.run(kernel_variant=EXPANDED), EXPANDED, f"{heads} heads {n} of {L}")


@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("w", [torch.float32, torch.bfloat16, torch.float16])
def test_types(cuda, kv, q, w):
    """Every mixture of cache, query and weight types; weights of another type are rounded to the expanded one (the
    reference takes them so)."""
    c = Case(cuda, "packed", [70, 33], [70, 20], kv=kv, q=q, w=w)
    c.W_UK, c.W_UV = (x.to(kv).to(x.dtype) for x in (c.W_UK, c.W_UV))
    for out in (torch.float32, torch.bfloat16, torch.float16):
        got = c.run(kernel_variant=EXPANDED, out_dtype=out)
        assert got.dtype == out
        c.check(got, EXPANDED, f"{kv} {q} {w} {out}")


@pytest.mark.parametrize("form", [PLAIN, ABSORBED])
@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.float32])
@pytest.mark.parametrize("q", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("w", [torch.float32, torch.bfloat16])
def test_types_of_the_other_forms(cuda, form, kv, q, w):
    """Every mixture that the plain and the absorbed form take, with 3 heads (no matrix instructions) and 32."""
    for heads in (3, 32):
        c = Case(cuda, "capacity", [70, 0, 33], [2, 1, 5], heads=heads, kv=kv, q=q, w=w, pad=1)
        full = c.run(kernel_variant=form, out_dtype=torch.float32)
        for out in (torch.float32, torch.bfloat16, torch.float16):
            got = c.run(kernel_variant=form, out_dtype=out)
            assert got.dtype == out
            # the merges of the two outputs may add in different orders: 2^-11 of the value, and one rounding
            assert ((got.float() - full).abs() <= (2.0 ** -11 + U.get(out, 0.0)) * full.abs() + 1e-4).all()
        assert_close(full.cpu().numpy(), c.reference()[0].numpy(), "bf16", f"{kv} {q} {w} {heads}")


def test_rotation_and_strides(cuda):
    """Queries rotated on the way equal queries rotated before; packed, sliced and oddly strided queries agree."""
    c = Case(cuda, "packed", [90, 40], [90, 11], heads=5, q=torch.float32)
    want = c.run(kernel_variant=EXPANDED)
    c.check(want, EXPANDED, "rotated on the way")
    pos = torch.cat([torch.arange(90), torch.arange(29, 40)]).to(cuda)
    x, y = c.q[..., 128:160], c.q[..., 160:]
    cs, sn = c.cos[pos][:, None], c.sin[pos][:, None]
    before = torch.cat([x * cs - y * sn, x * sn + y * cs], -1)
    kept = before.clone()
    args = (c.W_UK, c.W_UV, c.cos, c.sin, c.cfg)
    got = F.mla_prefill(c.layout.kv, c.q[..., :128].contiguous(), before, *args, **c.kw, kernel_variant=EXPANDED)
    assert torch.equal(before, kept)
    # a product contracted into an fma or not moves a rotated element by an fp32 rounding, which can move its 16-bit one
    assert (got - want).norm() <= 2.0 ** -8 * want.norm()
    wide = torch.zeros(101, 7, 193, device=cuda)  # rows that are no multiple of 16 bytes
    wide[:, 1:6, 1:] = c.q
    view = wide[:, 1:6, 1:]
    got = F.mla_prefill(c.layout.kv, view[..., :128], view[..., 128:], *args, **c.kw, rotate_q=True, kernel_variant=EXPANDED)
    assert torch.equal(got, want)
    turned = c.q.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    got = F.mla_prefill(c.layout.kv, turned[..., :128], turned[..., 128:], *args, **c.kw, rotate_q=True,
                        kernel_variant=EXPANDED)
    assert torch.equal(got, want)


@pytest.mark.parametrize("q", [torch.bfloat16, torch.float16])
def test_queries_by_alignment(cuda, q):
    """16-bit queries on 16, 8 and 2 bytes, and with strides that are no multiple of 16 bytes: the same numbers."""
    c = Case(cuda, "packed", [90, 40], [90, 11], heads=5, q=q)
    want = c.run(kernel_variant=EXPANDED)
    c.check(want, EXPANDED, f"{q}")
    kept = c.q
    for lead, pad in ((0, 0), (8, 0), (4, 0), (1, 0), (0, 4), (0, 1)):
        wide = torch.zeros(101 * 5 * (192 + pad) + lead, dtype=q, device=cuda)[lead:].view(101, 5, 192 + pad)
        wide[..., :192] = kept
        c.q = wide[..., :192]
        assert torch.equal(c.run(kernel_variant=EXPANDED), want), (lead, pad)


def test_unaligned_cache_and_weights(cuda):
    c = Case(cuda, "packed", [70, 33], [70, 20])
    want = c.run(kernel_variant=EXPANDED)
    for name in ("W_UK", "W_UV"):
        w = getattr(c, name)
        b = torch.zeros(w.numel() + 1, dtype=w.dtype, device=cuda)
        b[1:] = w.flatten()
        setattr(c, name, b[1:].view_as(w))
    b = torch.zeros(c.layout.kv.numel() + 1, dtype=c.layout.kv.dtype, device=cuda)
    b[1:] = c.layout.kv.flatten()
    c.layout.kv = b[1:].view_as(c.layout.kv)
    assert torch.equal(c.run(kernel_variant=EXPANDED), want)


@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("layout", ["capacity", "packed_capacity", "paged"])
@pytest.mark.parametrize("heads", [32, 128])
@pytest.mark.parametrize("aligned", [True, False])
def test_many_heads(cuda, heads, layout, kv, aligned):
    """The expansion's other tiles (few heads gather in its own workgroups), over caches that begin at any element."""
    c = Case(cuda, layout, [1, 63, 65, 200], [1, 5, 65, 30], heads=heads, kv=kv)
    if not aligned:
        b = torch.zeros(c.layout.kv.numel() + 1, dtype=torch.float32, device=cuda).to(kv)
        b.view(torch.uint8)[kv.itemsize:] = c.layout.kv.flatten().view(torch.uint8)
        c.layout.kv = b[1:].view_as(c.layout.kv)
    c.check(c.run(kernel_variant=EXPANDED), EXPANDED, f"{heads} {layout} {kv}")


@pytest.mark.parametrize("heads", [4, 32, 128])
def test_a_row_that_is_not_finite_by_size(cuda, heads):
    c = Case(cuda, "packed", [150, 80], [150, 80], heads=heads)
    want = c.run(kernel_variant=EXPANDED)
    c.layout.kv[101, 300], c.layout.kv[160, 7] = float("inf"), float("nan")
    got = c.run(kernel_variant=EXPANDED)
    assert torch.equal(got[:101], want[:101]) and torch.equal(got[150:160], want[150:160])
    assert not torch.isfinite(got[101:150]).any() and not torch.isfinite(got[160:]).any()


@pytest.mark.parametrize("form", [PLAIN, EXPANDED])
def test_rows_before_the_first_sequence(cuda, form):
    """Packed sequences that begin past the cache's first rows, which hold NaN."""
    c = Case(cuda, "packed", [70, 130], [70, 20])
    lead = torch.full((200, 576), float("nan"), dtype=c.layout.kv.dtype, device=cuda)
    want = c.run(kernel_variant=form)
    c.layout.kv = torch.cat([lead, c.layout.kv])
    c.kw["seq_offsets"] = c.kw["seq_offsets"] + 200
    got = c.run(kernel_variant=form)
    c.check(got, form, "rows before the first sequence")
    # the longer cache may cut its keys into more parts, whose sums are taken in another order
    assert form == EXPANDED or torch.equal(got, want)


@pytest.mark.parametrize("form", [PLAIN, EXPANDED, ABSORBED])
def test_broadcast_queries(cuda, form):
    """One query row for all tokens and heads, and one per token or head."""
    c = Case(cuda, "capacity", [40, 9], [3, 4], heads=16)
    for shape in ((1, 1), (7, 1), (1, 16)):
        one = c.q[:shape[0], :shape[1]].clone().expand(7, 16, 192)
        c.q = one.contiguous()
        want = c.run(kernel_variant=form)
        c.check(want, form, f"broadcast {shape}")
        c.q = one
        assert torch.equal(c.run(kernel_variant=form), want)
        c.q = one.contiguous()


@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float32])
def test_no_rows_at_all(cuda, kv):
    cfg, q = config(4), torch.randn(6, 4, 192, device=cuda)
    W = torch.zeros(512, 512, device=cuda, dtype=kv)
    t = torch.zeros(8, 32, device=cuda)
    got = F.mla_prefill(torch.zeros(2, 0, 576, device=cuda, dtype=kv), q[..., :128], q[..., 128:], W, W, t, t, cfg)
    assert got.shape == (6, 4, 128) and (got == 0).all()
    off = torch.zeros(3, dtype=torch.int32, device=cuda)
    got = F.mla_prefill(torch.zeros(0, 576, device=cuda, dtype=kv), q[..., :128], q[..., 128:], W, W, t, t, cfg,
                        seq_offsets=off, q_offsets=off)
    assert (got == 0).all()
    got = F.mla_prefill(torch.zeros(2, 8, 576, device=cuda, dtype=kv), q[:0, :, :128], q[:0, :, 128:], W, W, t, t, cfg)
    assert got.shape == (0, 4, 128)


@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("L", [50, 96])
def test_absorbed_over_equal_regions(cuda, L, kv):
    """Identity block tables: regions that are whole blocks of 32 rows, and one block each where they are not."""
    c = Case(cuda, "uniform", [L, L, L], [5, 5, 5], heads=16, kv=kv, q=torch.float32)
    c.check(c.run(kernel_variant=ABSORBED), ABSORBED, f"{kv} {L}")


def test_offsets_past_32_bits(cuda):
    """A cache whose expanded keys pass 2^31 elements and 2^32 bytes, in two groups of heads, against the absorbed form
    (both within 1e-2 of the exact result normwise, so within 2e-2 of each other)."""
    heads, L = 128, 140000
    cfg = config(heads)
    g = torch.Generator(device=cuda).manual_seed(1)
    kv = torch.randn(1, L, 576, generator=g, device=cuda).bfloat16()
    W_UK, W_UV = (w.to(cuda) for w in weights(heads, torch.bfloat16, 2))
    cos, sin = (t.to(cuda) for t in tables(L))
    q = torch.randn(3, heads, 192, generator=g, device=cuda)
    run = lambda form: F.mla_prefill(kv, q[..., :128], q[..., 128:], W_UK, W_UV, cos, sin, cfg, kernel_variant=form).double()
    a, b = run(ABSORBED), run(EXPANDED)
    assert (a - b).norm() <= 2e-2 * a.norm()


@pytest.mark.parametrize("form", [PLAIN, EXPANDED, ABSORBED])
def test_lengths_outside_their_regions(cuda, form):
    """A length beyond its region counts as the region, a negative one as none; as where they say so themselves."""
    c = Case(cuda, "capacity", [96, 96, 40], [3, 9, 5], heads=16)
    cap = c.layout.kv.shape[1]
    c.layout.kv[0, 96:] = c.layout.kv[0, :cap - 96]
    for given, meant in (([cap, 96, 40], [cap + 1000, 96, 40]), ([96, 0, 40], [96, -5, 40]), ([96, 96, 0], [96, 96, -2 ** 31])):
        out = []
        for lens in (given, meant):
            c.kw["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=cuda)
            out.append(c.run(kernel_variant=form))
        assert torch.isfinite(out[0]).all() and torch.equal(*out), (given, meant)


@pytest.mark.parametrize("form", [PLAIN, EXPANDED, ABSORBED])
def test_blocks_outside_the_pool(cuda, form):
    """Block numbers past the pool or below it take its last or first block (a row of which the sequence has)."""
    c = Case(cuda, "paged", [40, 64], [3, 9], heads=16, block=64)
    table, blocks = c.kw["block_table"], c.layout.kv.shape[0] // 64
    c.layout.kv.copy_(torch.randn(c.layout.kv.shape, generator=torch.Generator().manual_seed(4)).to(c.layout.kv.dtype))
    out = []
    for ids in ([blocks - 1, 0], [blocks + 5, -7], [2 ** 31 - 1, -2 ** 31]):
        table[:, 0] = torch.tensor(ids, dtype=torch.int32)
        out.append(c.run(kernel_variant=form))
    assert torch.isfinite(out[0]).all() and torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])


@pytest.mark.parametrize("form", [PLAIN, EXPANDED, ABSORBED])
def test_tables_that_end_early(cuda, form):
    """Positions past the tables take their last row: keys' and queries'."""
    c = Case(cuda, "capacity", [100, 30], [20, 4], heads=16)
    cos, sin = c.cos, c.sin
    ends = torch.arange(cos.shape[0], device=cuda).clamp(max=69)
    c.cos, c.sin = cos[ends], sin[ends]
    ref = c.reference()
    c.cos, c.sin = cos[:70].contiguous(), sin[:70].contiguous()
    got = c.run(kernel_variant=form)
    assert_close(got.double().cpu().numpy(), ref[0].numpy(), "bf16", "short tables")


@pytest.mark.parametrize("rows,new,prefix", [([2000], [3], [1500]), ([6300], [200], None), ([6300], [200], [6250]),
                                             ([64 * 97, 5], [130, 5], None)])
def test_long_caches(cuda, rows, new, prefix):
    """Parts of the keys under a prefix mask, and both orders of the workgroups. (A term of an output passes at most
    6300 / 16 additions of an instruction's 16 keys, one of a sum of weights 6300 / 8 of a lane's: the bound's fp32
    part, for 1000, holds.)"""
    for heads in (2, 8):
        c = Case(cuda, "capacity", rows, new, heads=heads, prefix=prefix)
        c.check(c.run(kernel_variant=EXPANDED), EXPANDED, f"{rows} {heads}")


def test_pages_cut_at_max_seq_rows(cuda):
    """Regions of whole and of cut blocks: rows past max_seq_rows are not seen."""
    c = Case(cuda, "paged", [130, 70, 200], [5, 3, 8], heads=16, block=48)
    held = c.rows
    for cut in (144, 100):
        c.rows = [r[:cut] for r in held]
        for form in (PLAIN, EXPANDED, ABSORBED):
            c.check(c.run(kernel_variant=form, max_seq_rows=cut), form, f"cut at {cut}")


def test_two_streams_at_once(cuda):
    """Two prompts on two streams, several times over: each has its own workspace."""
    cases = [Case(cuda, "packed", [700, 64], [700, 64], heads=16, seed=s) for s in (1, 2)]
    want = [c.run(kernel_variant=EXPANDED) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(5):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(c.run(kernel_variant=EXPANDED))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in (0, 1) for g in got[i])


def test_inputs_are_left_as_they_were(cuda):
    c = Case(cuda, "paged", ODD_ROWS, [1, 5, 8, 3, 1, 7], heads=16)
    tensors = [c.layout.kv, c.q, c.W_UK, c.W_UV, c.cos, c.sin, *[t for t in c.kw.values() if torch.is_tensor(t)]]
    before = [t.clone() for t in tensors]
    for form in (PLAIN, EXPANDED, ABSORBED):
        c.run(kernel_variant=form)
    for t, b in zip(tensors, before):
        assert torch.equal(t.view(torch.uint8) if t.is_floating_point() else t, b.view(torch.uint8) if b.is_floating_point() else b)


def test_c_entry_and_its_workspaces(cuda):
    """The C entry with a workspace of just its size at an odd address, with none, and twice over the same one."""
    import ctypes

    from latent_attn import capi

    lib = capi.load()
    c = Case(cuda, "capacity", [70, 9, 130], [20, 9, 1], heads=16, q=torch.float32)
    for form in (PLAIN, EXPANDED, ABSORBED):
        want = c.run(kernel_variant=form)
        out = torch.empty_like(want)
        q_nope, q_rope = c.q[..., :128].contiguous(), c.q[..., 128:].contiguous()
        a = capi.PrefillArgs(kv_cache=c.layout.kv.data_ptr(), kv_dtype=capi.LA_DTYPE_BF16, num_seqs=3,
                             seq_len=c.layout.kv.shape[1], total_rows=3 * c.layout.kv.shape[1],
                             seq_lens=c.kw["seq_lens"].data_ptr(), q_offsets=c.kw["q_offsets"].data_ptr(), tokens=30,
                             q_nope=q_nope.data_ptr(), q_rope=q_rope.data_ptr(), q_dtype=capi.LA_DTYPE_F32, rotate_q=1,
                             W_UK=c.W_UK.data_ptr(), w_uk_dtype=capi.LA_DTYPE_BF16, W_UV=c.W_UV.data_ptr(),
                             w_uv_dtype=capi.LA_DTYPE_BF16, rope_cos=c.cos.data_ptr(), rope_sin=c.sin.data_ptr(),
                             rope_rows=c.cos.shape[0], output=out.data_ptr(), out_dtype=capi.LA_DTYPE_F32,
                             cfg=capi.config(c.cfg), kernel_variant=form)
        stream = torch.cuda.current_stream().cuda_stream
        need = lib.la_mla_prefill_workspace_size(ctypes.byref(a))
        ws = torch.full((need + 64,), 255, dtype=torch.uint8, device=cuda)
        for at in (0, 16, 16):
            out.fill_(float("nan"))
            a.workspace, a.workspace_bytes = ws.data_ptr() + at, need
            assert lib.la_mla_prefill(ctypes.byref(a), stream) == capi.LA_SUCCESS
            assert torch.equal(out, want), (form, at)
        assert (ws[need + 16:] == 255).all()
        out.fill_(float("nan"))
        a.workspace, a.workspace_bytes = None, 0
        assert lib.la_mla_prefill(ctypes.byref(a), stream) == capi.LA_SUCCESS
        assert torch.equal(out, want), form


@pytest.mark.parametrize("block", [1, 16, 48, 100])
def test_page_sizes(cuda, block):
    """Pages that end inside a tile of keys, and single rows."""
    c = Case(cuda, "paged", ODD_ROWS, ODD_NEW, block=block)
    c.check(c.run(kernel_variant=EXPANDED), EXPANDED, f"block {block}")


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_a_token_does_not_see_does_not_reach_it(cuda, bad):
    """Rows behind a token that hold NaN or infinities leave it as it was; the tokens that see them get NaN or
    infinities (nothing finite), in every head."""
    c = Case(cuda, "packed", [150, 80], [150, 80])
    want = c.run(kernel_variant=EXPANDED)
    c.layout.kv[101] = bad  # a row of the first sequence
    got = c.run(kernel_variant=EXPANDED)
    assert torch.equal(got[:101], want[:101]) and torch.equal(got[150:], want[150:])
    assert not torch.isfinite(got[101:150]).any()


def test_large_scores(cuda):
    """Scores of thousands: the running maximum rises often, and by much."""
    c = Case(cuda, "packed", [300, 64], [300, 64], scale=1.0)
    c.q *= 64
    c.q_type = torch.bfloat16
    ref = c.reference()
    got = c.run(kernel_variant=EXPANDED).double().cpu()
    assert torch.isfinite(got).all()
    # a rounded key moves a score of hundreds by more than one: only rows whose first weight is safe are compared
    out, mass, size = ref
    top = (got - out).abs().amax(-1)
    safe = torch.expm1(2 * 2 * 2.0 ** -8 * size) < 0.5
    assert (top[safe] <= 2 * mass.amax(-1)[safe]).all()


def test_splits_equal_one_part(cuda):
    """One token tile over many keys runs in parts of the keys, joined; the same call in a large batch does not."""
    one = Case(cuda, "uniform", [2000], [3], heads=2, seed=5)
    got = one.run(kernel_variant=EXPANDED)
    one.check(got, EXPANDED, "parts")


def test_auto_form_and_large_head_count(cuda):
    for rows, new in (([400, 90], [3, 1]), ([400, 90], [300, 90])):
        c = Case(cuda, "paged", rows, new, heads=128)
        c.check(c.run(), ABSORBED, "auto")


def test_other_dims(cuda):
    for kv in (torch.bfloat16, torch.float32):
        c = Case(cuda, "packed", [50, 20], [50, 3], heads=3, kv=kv, q=torch.float32, dims=(96, 40, 24, 56))
        c.check(c.run(), PLAIN, "other dims")


def test_max_seq_rows(cuda):
    """A capacity cache whose regions are cut at max_seq_rows gives the same where no sequence is longer."""
    c = Case(cuda, "capacity", [50, 64, 10], [50, 5, 10], heads=16)
    for form in (PLAIN, EXPANDED, ABSORBED):
        want = c.run(kernel_variant=form)
        got = c.run(kernel_variant=form, max_seq_rows=64)
        c.check(got, form, "max_seq_rows")
        # (the absorbed form's decode plan cuts the region, so its sums run in another order)
        assert form == ABSORBED or torch.equal(got, want)


def test_other_stream_and_repeat(cuda):
    c = Case(cuda, "packed", ODD_ROWS, ODD_NEW)
    want = c.run(kernel_variant=EXPANDED)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [c.run(kernel_variant=EXPANDED) for _ in range(3)]
    torch.cuda.synchronize()
    for g in got:
        assert torch.equal(g, want)


@pytest.mark.parametrize("form", [PLAIN, EXPANDED, ABSORBED])
def test_captured(cuda, form):
    """A captured call replayed on other inputs and offsets (a padded batch), with eager work between the replays."""
    c = Case(cuda, "capacity", [50, 64, 10], [20, 5, 10], heads=16, pad=10)
    c.run(kernel_variant=form)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.run(kernel_variant=form)
    for seed, new in ((3, [20, 5, 10]), (4, [1, 40, 4]), (5, [0, 0, 1])):
        g = torch.Generator().manual_seed(seed)
        c.q.copy_(torch.randn(c.q.shape, generator=g).to(c.q.dtype))
        at = [0, new[0], new[0] + new[1], sum(new)]
        c.kw["q_offsets"].copy_(torch.tensor(at, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        eager = c.run(kernel_variant=form)
        torch.cuda.synchronize()
        assert torch.equal(got, eager)
        assert (got[sum(new):] == 0).all()


@pytest.mark.parametrize("heads,cap", [(2, 2048), (64, 256)])
def test_captured_by_size(cuda, heads, cap):
    """Parts of the keys and their join, and the expansion in a launch of its own, in a graph; lengths that change."""
    c = Case(cuda, "capacity", [cap - 40, 70], [3, 60], heads=heads)
    c.run(kernel_variant=EXPANDED)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.run(kernel_variant=EXPANDED)
    c.layout.kv.copy_(torch.randn(c.layout.kv.shape, generator=torch.Generator().manual_seed(7)).to(c.layout.kv.dtype))
    for lens, new in (([cap - 40, 70], [3, 60]), ([1, cap], [1, 62]), ([0, 65], [60, 3]), ([64, 128], [0, 63])):
        c.kw["seq_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        c.kw["q_offsets"].copy_(torch.tensor([0, new[0], sum(new)], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        eager = c.run(kernel_variant=EXPANDED)
        torch.cuda.synchronize()
        assert torch.equal(got, eager) and torch.isfinite(got).all()


def test_prompt_then_decode(cuda):
    """append_kv of a prompt, its attention, then a drafted pair of tokens and a single one: the last token's row is
    the decode step's."""
    cfg = config(16)
    B, cap, T = 3, 256, 70
    g = torch.Generator().manual_seed(2)
    W_UK, W_UV = (x.to(cuda) for x in weights(16, torch.bfloat16, 3))
    cos, sin = (x.to(cuda) for x in tables(cap))
    kv = torch.full((B, cap, 576), float("nan"), dtype=torch.bfloat16, device=cuda)
    lens = torch.zeros(B, dtype=torch.int32, device=cuda)
    rows = torch.randn(B, T + 3, 576, generator=g).to(torch.bfloat16).to(cuda)
    q = torch.randn(B, T + 3, 16, 192, generator=g).to(cuda)
    at = 0
    for n in (T, 2, 1):
        new = rows[:, at:at + n]
        F.append_kv(kv, lens, new[..., :512].contiguous(), new[..., 512:].contiguous(), cfg)
        at += n
        mine = q[:, at - n:at].reshape(B * n, 16, 192)
        got = F.mla_prefill(kv, mine[..., :128], mine[..., 128:], W_UK, W_UV, cos, sin, cfg, seq_lens=lens, rotate_q=True)
        ref = reference([r[:at] for r in as_double(rows)], as_double(mine[..., :128]), as_double(mine[..., 128:]),
                        as_double(W_UK), as_double(W_UV), as_double(cos), as_double(sin), [n] * B, None, True)
        assert_close(got.double().cpu().numpy(), ref[0].numpy(), "bf16", f"{n} tokens at {at}")
        assert lens.tolist() == [at] * B
    x, y = mine[..., 128:160], mine[..., 160:]
    cs, sn = cos[at - 1], sin[at - 1]
    turned = torch.cat([x * cs - y * sn, x * sn + y * cs], -1).contiguous()
    step = F.mla_decode(kv, mine[..., :128].contiguous(), turned, W_UK, W_UV, cos, sin, cfg, seq_lens=lens)
    assert_close(got.cpu().numpy(), step.double().cpu().numpy(), "bf16", "the decode step")
