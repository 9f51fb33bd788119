"""GPU parity of functional.expand_prefix and functional.mla_decode_shared
against the 64-bit reference of tests/prompt_cases.py, and against
functional.mla_decode over caches that hold the prefix themselves."""

from __future__ import annotations

import pytest
import torch

from conftest import assert_close
from prompt_cases import U, Layout, as_double, reference, rotate, tables, weights

from latent_attn import MLAConfig
from latent_attn import functional as F

pytestmark = pytest.mark.gpu

AUTO, LATENT, EXPANDED = 0, 1, 2


def config(heads, dc=512, dn=128, d_r=64, dv=128):
    return MLAConfig(5120, dc, dn, d_r, heads, dv)


@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("rows,heads", [(1, 1), (64, 3), (65, 8), (200, 17), (700, 2)])
def test_expand(cuda, rows, heads, kv):
    """K, V and rope keys, element by element: sums of 512 products in fp32 (each off by at most 512 2^-24 of the sum
    of magnitudes) and one rounding; zeros past the last row."""
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, 576, generator=g).to(kv).to(cuda)
    model = torch.float16 if kv == torch.float16 else torch.bfloat16
    W_UK, W_UV = (w.to(cuda) for w in weights(heads, model, 4))
    cos, sin = (t.to(cuda) for t in tables(rows))
    p = F.expand_prefix(x, W_UK, W_UV, cos, sin, config(heads))
    c, r = as_double(x)[:, :512], as_double(x)[:, 512:]
    for got, W, axis in ((p.k_nope, W_UK, 0), (p.v, W_UV, 0)):
        got = as_double(got.reshape(-1, heads, 128))
        want = (c @ as_double(W).T).view(rows, heads, 128)
        size = (c.abs() @ as_double(W).abs().T).view(rows, heads, 128)
        assert ((got[:rows] - want).abs() <= U[model] * want.abs() + 512 * 2.0 ** -24 * size + 2.0 ** -25).all()
        assert (got[rows:] == 0).all()
    got = as_double(p.k_rope.reshape(-1, 64))
    want = rotate(r, as_double(cos), as_double(sin))
    assert ((got[:rows] - want).abs() <= U[model] * want.abs() + 4 * 2.0 ** -24 * r.abs().amax()).all()
    assert (got[rows:] == 0).all()


class Case:
    def __init__(self, cuda, prefix, own, heads=16, kv=torch.bfloat16, layout="paged", seed=1, dims=(512, 128, 64, 128),
                 model=None):
        dc, dn, d_r, dv = dims
        self.cfg, self.kv_type = config(heads, dc, dn, d_r, dv), kv
        g = torch.Generator().manual_seed(seed)
        front = torch.randn(prefix, dc + d_r, generator=g).to(kv).float()
        data = [torch.randn(n, dc + d_r, generator=g).to(kv).float() for n in own]
        self.layout = Layout(layout, data, kv, cuda, seed=seed)
        self.front = front.to(kv).to(cuda)
        self.rows = [torch.cat([front, d]).double() for d in data]
        model = model or (kv if kv in U else torch.float32 if kv == torch.float32 else torch.bfloat16)
        self.W_UK, self.W_UV = (w.to(cuda) for w in weights(heads, model, seed + 1, dc, dn, dv))
        self.cos, self.sin = (t.to(cuda) for t in tables(prefix + max(own), d_r))
        self.q_nope = torch.randn(len(own), heads, dn, generator=g).to(cuda)
        self.q_rope = torch.randn(len(own), heads, d_r, generator=g).to(cuda)

    def expand(self):
        return F.expand_prefix(self.front, self.W_UK, self.W_UV, self.cos, self.sin, self.cfg)

    def run(self, prefix=None, **kw):
        return F.mla_decode_shared(self.front if prefix is None else prefix, self.layout.kv, self.q_nope, self.q_rope,
                                   self.W_UK, self.W_UV, self.cos, self.sin, self.cfg, **self.layout.kw, **kw)

    def reference(self):
        return reference(self.rows, as_double(self.q_nope), as_double(self.q_rope), as_double(self.W_UK),
                         as_double(self.W_UV), as_double(self.cos), as_double(self.sin), [1] * len(self.rows))[0]

    def check(self, got, what):
        kind = "f32" if self.kv_type == torch.float32 else "bf16"
        assert_close(got.double().cpu().numpy(), self.reference().numpy(), kind, what)


@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("layout", ["packed", "capacity", "packed_capacity", "paged"])
@pytest.mark.parametrize("form", [LATENT, EXPANDED])
def test_layouts(cuda, layout, form, kv):
    c = Case(cuda, 150, [0, 1, 64, 65, 33], kv=kv, layout=layout)
    c.check(c.run(c.expand(), kernel_variant=form), f"{layout} {kv} {form}")


@pytest.mark.parametrize("layout", ["packed", "capacity", "paged"])
def test_f32(cuda, layout):
    c = Case(cuda, 150, [0, 1, 64, 65, 33], kv=torch.float32, layout=layout)
    c.check(c.run(), layout)


@pytest.mark.parametrize("form", [LATENT, EXPANDED])
@pytest.mark.parametrize("prefix", [1, 63, 64, 65, 1000])
@pytest.mark.parametrize("batch,heads", [(1, 16), (2, 128), (130, 8), (33, 3)])
def test_sizes(cuda, prefix, batch, heads, form):
    c = Case(cuda, prefix, [(11 * i) % 40 for i in range(batch)], heads=heads, layout="capacity")
    c.check(c.run(c.expand(), kernel_variant=form), f"{batch} x {prefix} x {heads}")


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
def test_output_types(cuda, out):
    c = Case(cuda, 100, [5, 0, 9])
    for form in (LATENT, EXPANDED):
        full = c.run(c.expand(), kernel_variant=form)
        got = c.run(c.expand(), kernel_variant=form, out_dtype=out)
        assert got.dtype == out and torch.equal(got, full.to(out))


def test_empty_prefix_and_empty_rows(cuda):
    c = Case(cuda, 0, [0, 7, 64], layout="capacity")
    got = c.run()
    c.check(got, "no prefix")
    assert (got[0] == 0).all()
    again = F.mla_decode(c.layout.kv, c.q_nope, c.q_rope, c.W_UK, c.W_UV, c.cos, c.sin, c.cfg, **c.layout.kw)
    assert torch.equal(got, again)
    c = Case(cuda, 90, [0, 0, 0], layout="paged")
    for form in (LATENT, EXPANDED):
        c.check(c.run(c.expand(), kernel_variant=form), "no own rows")


def test_equals_decode_over_whole_caches(cuda):
    c = Case(cuda, 200, [30, 1, 64, 100], heads=32, layout="capacity")
    cap = c.layout.kv.shape[1]
    whole = torch.cat([c.front.expand(4, -1, -1), c.layout.kv], 1).contiguous()
    lens = (c.layout.kw["seq_lens"] + 200).int()
    assert whole.shape[1] == 200 + cap
    step = F.mla_decode(whole, c.q_nope, c.q_rope, c.W_UK, c.W_UV, c.cos, c.sin, c.cfg, seq_lens=lens)
    for form in (LATENT, EXPANDED):
        got = c.run(c.expand(), kernel_variant=form)
        assert_close(got.double().cpu().numpy(), step.double().cpu().numpy(), "bf16", "decode over whole caches")


@pytest.mark.parametrize("form", [LATENT, EXPANDED])
def test_several_queries_per_sequence(cuda, form):
    """The C entry's queries_per_seq, on packed own rows and a caller's workspace, an odd address among them."""
    import ctypes

    from latent_attn import capi

    lib, heads, own, P = capi.load(), 16, [7, 0, 40], 100
    c = Case(cuda, P, own, heads=heads, layout="packed")
    g = torch.Generator().manual_seed(9)
    q_nope, q_rope = (torch.randn(6, heads, d, generator=g).to(cuda) for d in (128, 64))
    out = torch.empty(6, heads, 128, device=cuda)
    expanded = c.expand().expanded
    a = capi.SharedArgs(prefix=c.front.data_ptr(), prefix_len=P, expanded=expanded.data_ptr(), output=out.data_ptr(),
                        out_dtype=capi.LA_DTYPE_F32, kernel_variant=form)
    a.own = capi.DecodeArgs(kv_cache=c.layout.kv.data_ptr(), kv_dtype=capi.LA_DTYPE_BF16, total_rows=47, num_seqs=3,
                            seq_offsets=c.layout.kw["seq_offsets"].data_ptr(), queries_per_seq=2,
                            q_nope=q_nope.data_ptr(), q_rope=q_rope.data_ptr(), W_UK=c.W_UK.data_ptr(),
                            w_uk_dtype=capi.LA_DTYPE_BF16, W_UV=c.W_UV.data_ptr(), w_uv_dtype=capi.LA_DTYPE_BF16,
                            rope_cos=c.cos.data_ptr(), rope_sin=c.sin.data_ptr(), rope_rows=c.cos.shape[0],
                            cfg=capi.config(c.cfg))
    stream = torch.cuda.current_stream().cuda_stream
    need = lib.la_mla_decode_shared_workspace_size(ctypes.byref(a))
    ws = torch.full((need + 64,), 255, dtype=torch.uint8, device=cuda)
    ref = reference([r for r in c.rows for _ in range(2)], as_double(q_nope), as_double(q_rope), as_double(c.W_UK),
                    as_double(c.W_UV), as_double(c.cos), as_double(c.sin), [1] * 6)[0]
    for at in (0, 16):
        out.fill_(float("nan"))
        a.workspace, a.workspace_bytes = ws.data_ptr() + at, need
        assert lib.la_mla_decode_shared(ctypes.byref(a), stream) == capi.LA_SUCCESS
        assert_close(out.double().cpu().numpy(), ref.numpy(), "bf16", f"two queries, workspace + {at}")
    assert (ws[need + 16:] == 255).all()
    a.workspace, a.workspace_bytes = None, 0  # taken in the order of the stream
    assert lib.la_mla_decode_shared(ctypes.byref(a), stream) == capi.LA_SUCCESS
    assert_close(out.double().cpu().numpy(), ref.numpy(), "bf16", "own memory")


def test_a_row_that_is_not_finite(cuda):
    """An infinity or NaN in the prefix reaches every token, in one sequence's own rows that sequence's only."""
    for bad in (float("nan"), float("inf")):
        c = Case(cuda, 130, [5, 40, 0], layout="capacity")
        p = c.expand()
        want = c.run(p, kernel_variant=EXPANDED)
        c.layout.kv[1, 3] = bad
        got = c.run(p, kernel_variant=EXPANDED)
        assert not torch.isfinite(got[1]).any() and torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
        c = Case(cuda, 130, [5, 40, 0], layout="capacity")
        c.front[77] = bad
        assert not torch.isfinite(c.run(c.expand(), kernel_variant=EXPANDED)).any()


def test_tables_that_end_early(cuda):
    """Positions past the tables take their last row, as everywhere."""
    c = Case(cuda, 100, [30, 64, 7], layout="capacity")
    full_cos, full_sin = c.cos, c.sin
    for rows in (110, 60):
        c.cos, c.sin = full_cos[:rows].contiguous(), full_sin[:rows].contiguous()
        ends = torch.arange(full_cos.shape[0]).clamp(max=rows - 1)
        ref = reference(c.rows, as_double(c.q_nope), as_double(c.q_rope), as_double(c.W_UK), as_double(c.W_UV),
                        as_double(full_cos)[ends], as_double(full_sin)[ends], [1] * 3)[0]
        if rows == 60:  # the extension asks for a table over the prefix; the C entry clamps
            with pytest.raises(RuntimeError, match="need at least"):
                c.run()
            continue
        assert_close(c.run().double().cpu().numpy(), ref.numpy(), "bf16", "clamped tables")


@pytest.mark.parametrize("model", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kv", [torch.float16, torch.bfloat16, torch.float8_e4m3fn])
def test_weight_types(cuda, kv, model):
    c = Case(cuda, 150, [5, 0, 40], kv=kv, layout="capacity", model=model)
    for form in (LATENT, EXPANDED):
        c.check(c.run(c.expand(), kernel_variant=form), f"{kv} {model} {form}")


@pytest.mark.parametrize("kv", [torch.float16, torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("model", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16),
                                   (torch.float16, torch.bfloat16)])
@pytest.mark.parametrize("heads", [16, 32, 128])
def test_weights_of_two_types(cuda, kv, model, heads):
    """Absorption and projection weights of their own types, with heads that share their absorbed queries between the
    two steps and others; into a workspace that holds NaN."""
    c = Case(cuda, 150, [5, 0, 40], heads=heads, kv=kv, layout="capacity", model=torch.float32)
    c.W_UK, c.W_UV = c.W_UK.to(model[0]), c.W_UV.to(model[1])
    p = c.expand()
    for form in (LATENT, EXPANDED):
        for _ in range(2):
            junk = torch.full((64 << 20,), float("nan"), device=cuda)  # what the allocator gives out next
            del junk
            c.check(c.run(p, kernel_variant=form), f"{kv} {model} {form}")


def test_lengths_outside_their_regions(cuda):
    c = Case(cuda, 100, [64, 9], layout="capacity")
    cap = c.layout.kv.shape[1]
    c.layout.kv[0, 64:] = c.layout.kv[0, :cap - 64]
    p = c.expand()
    for form in (LATENT, EXPANDED):
        for given, meant in (([cap, 9], [cap + 1, 9]), ([64, 0], [64, -3])):
            out = []
            for lens in (given, meant):
                c.layout.kw["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=cuda)
                out.append(c.run(p, kernel_variant=form))
            assert torch.isfinite(out[0]).all() and torch.equal(*out)


@pytest.mark.parametrize("form", [LATENT, EXPANDED])
def test_two_streams_at_once(cuda, form):
    """Two batches behind one expanded prefix, on two streams."""
    cases = [Case(cuda, 500, [20, 0, 40], heads=32, layout="capacity", seed=s) for s in (1, 2)]
    p = cases[0].expand()
    cases[1].W_UK, cases[1].W_UV = cases[0].W_UK, cases[0].W_UV
    want = [c.run(p, kernel_variant=form) for c in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[], []]
    for _ in range(5):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(c.run(p, kernel_variant=form))
    torch.cuda.synchronize()
    # few query rows: two halves of a row are added into zeros with atomics, in either order the same sum
    assert all(torch.equal(g, want[i]) for i in (0, 1) for g in got[i])


def test_other_dims(cuda):
    for kv in (torch.bfloat16, torch.float32):
        c = Case(cuda, 70, [5, 0, 30], heads=3, kv=kv, layout="packed", dims=(96, 40, 24, 56))
        c.check(c.run(), "other dims")
    with pytest.raises(RuntimeError, match="expand_prefix"):
        c.expand()


@pytest.mark.parametrize("form", [LATENT, EXPANDED])
def test_captured(cuda, form):
    c = Case(cuda, 300, [5, 20, 60], layout="capacity")
    p = c.expand()
    c.run(p, kernel_variant=form)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.run(p, kernel_variant=form)
    for seed, lens in ((3, [5, 20, 60]), (4, [0, 60, 1]), (5, [0, 0, 0])):
        g = torch.Generator().manual_seed(seed)
        c.layout.kv.copy_(torch.randn(c.layout.kv.shape, generator=g).to(c.layout.kv.dtype))
        c.q_nope.copy_(torch.randn(c.q_nope.shape, generator=g))
        c.layout.kw["seq_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        eager = c.run(p, kernel_variant=form)
        torch.cuda.synchronize()
        # few query rows: two halves of a row are added into zeros with atomics, in either order the same sum
        assert torch.equal(got, eager)


@pytest.mark.parametrize("rows,heads", [(130, 16), (700, 128)])
def test_captured_with_its_expansion(cuda, rows, heads):
    """A prefix that is expanded and read in one graph, replayed over other rows, with eager work between the replays."""
    c = Case(cuda, rows, [5, 20, 60], heads=heads, layout="capacity")
    run = lambda: c.run(c.expand(), kernel_variant=EXPANDED)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in (3, 4, 5):
        g = torch.Generator().manual_seed(seed)
        c.front.copy_(torch.randn(c.front.shape, generator=g).to(c.front.dtype))
        c.W_UV.copy_(torch.randn(c.W_UV.shape, generator=g) / 22)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        eager = run()
        torch.cuda.synchronize()
        assert torch.equal(got, eager)


def test_a_batch_served(cuda):
    """A server's round: the prefix expanded once, then every sequence's question appended and attended, and single
    tokens after it; each against the reference."""
    heads, P, B = 16, 130, 4
    cfg = config(heads)
    g = torch.Generator().manual_seed(6)
    W_UK, W_UV = (w.to(cuda) for w in weights(heads, torch.bfloat16, 7))
    cos, sin = (t.to(cuda) for t in tables(P + 64))
    front = torch.randn(P, 576, generator=g).to(torch.bfloat16).to(cuda)
    prefix = F.expand_prefix(front, W_UK, W_UV, cos, sin, cfg)
    kv = torch.full((B, 64, 576), float("nan"), dtype=torch.bfloat16, device=cuda)
    lens = torch.zeros(B, dtype=torch.int32, device=cuda)
    held = [as_double(front) for _ in range(B)]
    for _ in range(4):
        new = torch.randn(B, 1, 576, generator=g).to(torch.bfloat16).to(cuda)
        F.append_kv(kv, lens, new[..., :512].contiguous(), new[..., 512:].contiguous(), cfg)
        held = [torch.cat([h, as_double(n)]) for h, n in zip(held, new)]
        q_nope = torch.randn(B, heads, 128, generator=g).to(cuda)
        q_rope = torch.randn(B, heads, 64, generator=g).to(cuda)
        ref = reference(held, as_double(q_nope), as_double(q_rope), as_double(W_UK), as_double(W_UV), as_double(cos),
                        as_double(sin), [1] * B)[0]
        for form in (LATENT, EXPANDED):
            got = F.mla_decode_shared(prefix, kv, q_nope, q_rope, W_UK, W_UV, cos, sin, cfg, seq_lens=lens,
                                      kernel_variant=form)
            assert_close(got.double().cpu().numpy(), ref.numpy(), "bf16", "served")
