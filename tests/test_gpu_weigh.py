"""GPU parity of functional.weigh_kv (la_weigh_kv) against the 64-bit reference of tests/draft_cases.py, within the
bound derived there."""

from __future__ import annotations

import ctypes

import pytest
import torch

from draft_cases import room, weigh_reference, weight_places
from prompt_cases import Layout, as_double, tables, weights

from latent_attn import MLAConfig, capi
from latent_attn import functional as F

pytestmark = pytest.mark.gpu

AUTO, PLAIN, MFMA = 0, 1, 2


class Case:
    def __init__(self, cuda, layout, rows, n=1, heads=16, kv=torch.bfloat16, q=torch.bfloat16, w=None, rotate_q=True,
                 block=64, seed=1, dims=(512, 128, 64), data=None, scale=1.0):
        dc, dn, d_r = dims
        self.cfg = MLAConfig(5120, dc, dn, d_r, heads, 128)
        g = torch.Generator().manual_seed(seed)
        data = data or [(torch.randn(m, dc + d_r, generator=g) * scale).to(kv).float() for m in rows]
        self.layout = Layout(layout, data, kv, cuda, block=block, seed=seed)
        self.rows = [d.double() for d in data]
        self.q = torch.randn(len(rows) * n, heads, dn + d_r, generator=g).to(q).to(cuda)
        w = w or (kv if kv in (torch.float16, torch.bfloat16, torch.float32) else torch.bfloat16)
        self.W_UK = weights(heads, w, seed + 1, dc, dn, 128)[0].to(cuda)
        cos, sin = tables(max(rows + [1]), d_r)
        self.cos, self.sin = cos.to(cuda), sin.to(cuda)
        self.rotate_q, self.dn, self.n = rotate_q, dn, n
        self.weights = torch.rand(*room(self.layout), generator=g).to(cuda)

    def run(self, weights=None, **kw):
        kw = {**self.layout.kw, "rotate_q": self.rotate_q, **kw}
        F.weigh_kv(self.weights if weights is None else weights, self.layout.kv, self.q[..., :self.dn], self.q[..., self.dn:],
                   self.W_UK, self.cos, self.sin, self.cfg, **kw)

    def reference(self):
        q = as_double(self.q)
        return weigh_reference(self.rows, q[..., :self.dn], q[..., self.dn:], as_double(self.W_UK), as_double(self.cos),
                               as_double(self.sin), self.n, self.rotate_q)

    def check(self, variant=AUTO, what="", pieces=1):
        """From zeros, within the bound; on top of other weights, the same sum; nothing outside the sequences' rows.
        pieces: sums that the call adds to a weight one after another (4096 rows of tokens and heads at most in each)."""
        zero = torch.full_like(self.weights, 7.0)
        places = [weight_places(self.layout, s, r.shape[0]) for s, r in enumerate(self.rows)]
        inside = torch.cat(places) if places else torch.zeros(0, dtype=torch.long)
        zero.view(-1)[inside.to(zero.device)] = 0
        start = self.weights.clone()
        self.run(zero, kernel_variant=variant)
        self.run(kernel_variant=variant)
        got, more = zero.cpu().double().view(-1), self.weights.cpu().view(-1)
        for s, (at, w, b, norm) in enumerate(zip(places, *self.reference())):
            off = (got[at] - w).abs() - b
            assert (off <= 0).all(), f"{what} sequence {s}: {off.max():.3e} over the bound"
            if w.norm() > 0:
                off = float((got[at] - w).norm() / w.norm())
                assert off <= norm, f"{what} {s}: normwise {off:.3e}"
        outside = torch.ones(got.numel(), dtype=torch.bool)
        outside[inside] = False
        assert (got[outside] == 7).all()
        first = start.cpu().view(-1)
        assert torch.equal(more[outside], first[outside])
        # The weights are positive, so every partial sum is below the whole and its rounding below 2^-24 of that
        # (1 + 2^-20 for the roundings before it). P pieces make P such sums on top of other weights and P - 1 from
        # zero (the first is exact): 2 P - 1 together, and one piece is given 2.
        want = first[inside].double() + got[inside]
        assert ((more[inside].double() - want).abs() <= max(2, 2 * pieces - 1) * (1 + 2.0 ** -20) * 2.0 ** -24 * want).all()


@pytest.mark.parametrize("layout", ["uniform", "capacity", "packed", "packed_capacity", "paged"])
@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn])
@pytest.mark.parametrize("variant", [AUTO, PLAIN])
def test_by_layout_and_type(cuda, layout, kv, variant):
    rows = [70] * 3 if layout == "uniform" else [1, 70, 131, 32, 300]
    Case(cuda, layout, rows, heads=16, kv=kv, q=torch.float32).check(variant, f"{layout} {kv}")


@pytest.mark.parametrize("n", [1, 2, 5, 31, 64, 100])
@pytest.mark.parametrize("heads", [1, 3, 16, 40, 128])
def test_windows(cuda, n, heads):
    """Windows shorter and longer than their sequences (whose first tokens then see nothing)."""
    if n * heads > 2000:
        pytest.skip("the 64-bit reference is slow there")
    Case(cuda, "paged", [n + 90, n, max(n - 1, 1), 1, 64, 257], n, heads=heads, block=32, seed=n).check(AUTO, f"{n} {heads}")


@pytest.mark.parametrize("q", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rotate_q", [False, True])
def test_queries(cuda, q, rotate_q):
    for variant in (AUTO, PLAIN):
        Case(cuda, "capacity", [40, 100], 3, q=q, rotate_q=rotate_q).check(variant, f"{q} {rotate_q}")


@pytest.mark.parametrize("w", [torch.float32, torch.float16, torch.bfloat16])
def test_weights_of_every_type(cuda, w):
    Case(cuda, "capacity", [40, 100], 2, heads=32, w=w, q=torch.float32).check(AUTO, str(w))


@pytest.mark.parametrize("dims,heads", [((64, 32, 16), 5), ((96, 40, 6), 2), ((1024, 64, 128), 1)])
def test_other_head_shapes(cuda, dims, heads):
    Case(cuda, "packed_capacity", [5, 60, 77], 4, heads=heads, kv=torch.float32, q=torch.float32, dims=dims).check()


@pytest.mark.parametrize("scale", [8.0, 1 / 64])
@pytest.mark.parametrize("variant", [AUTO, PLAIN])
def test_scores_far_apart_and_all_alike(cuda, scale, variant):
    c = Case(cuda, "capacity", [400, 100], 2, q=torch.float32, scale=scale)
    c.check(variant, str(scale))


@pytest.mark.parametrize("block", [1, 7, 16, 48])
@pytest.mark.parametrize("heads", [16, 128])
def test_block_sizes(cuda, block, heads):
    Case(cuda, "paged", [100, 33, 64, 31, 5], 2, heads=heads, block=block).check(MFMA, block)


@pytest.mark.parametrize("variant", [AUTO, PLAIN])
@pytest.mark.parametrize("q", [torch.float32, torch.bfloat16])
def test_queries_out_of_line(cuda, variant, q):
    """Views whose elements are not aligned to whole vectors, by token, head or address."""
    for pad, skip in ((1, 0), (4, 1), (3, 2)):
        c = Case(cuda, "capacity", [150, 64, 300], 6, q=q, seed=pad)
        wide = torch.zeros(*c.q.shape[:2], c.q.shape[2] + pad, dtype=q, device=cuda)
        wide[..., skip:skip + c.q.shape[2]] = c.q
        c.q = wide[..., skip:skip + c.q.shape[2]]
        c.check(variant, (pad, skip))


# more (token, head) rows than one piece of the call takes
@pytest.mark.parametrize("n,heads,pieces", [(50, 128, 2), (300, 40, 3), (129, 33, 2)])
def test_pieces_of_tokens(cuda, n, heads, pieces):
    Case(cuda, "capacity", [n + 37, n, 20], n, heads=heads, kv=torch.float16).check(MFMA, (n, heads), pieces)


def test_pieces_of_sequences(cuda):
    """More room for scores than the call takes at once: in pieces of 128 sequences; each as on its own."""
    count, region, heads = 200, 8192, 128
    g = torch.Generator(device=cuda).manual_seed(3)
    cfg = MLAConfig(5120, 512, 128, 64, heads, 128)
    kv = torch.zeros(count, region, 576, dtype=torch.float8_e4m3fn, device=cuda)
    kv[:, :120] = torch.randn(count, 120, 576, generator=g, device=cuda).to(torch.float8_e4m3fn)
    lens = torch.randint(1, 121, (count,), generator=g, device=cuda, dtype=torch.int32)
    q = torch.randn(count, heads, 192, generator=g, device=cuda).bfloat16()
    W_UK = weights(heads, torch.bfloat16, 5, 512, 128, 128)[0].to(cuda)
    cos, sin = (x.to(cuda) for x in tables(region, 64))
    w = torch.zeros(count, region, device=cuda)
    F.weigh_kv(w, kv, q[..., :128], q[..., 128:], W_UK, cos, sin, cfg, seq_lens=lens, rotate_q=True)
    for s in (0, 1, 127, 128, 129, 199):
        n = int(lens[s])
        alone = torch.zeros(1, region, device=cuda)
        F.weigh_kv(alone, kv[s:s + 1], q[s:s + 1, :, :128], q[s:s + 1, :, 128:], W_UK, cos, sin, cfg, seq_lens=lens[s:s + 1],
                   rotate_q=True)
        # two orders of the same fp32 sums of 128 terms: 128 half steps each
        assert ((alone[0, :n] - w[s, :n]).abs() <= 256 * 2.0 ** -24 * w[s, :n]).all()
        assert abs(float(w[s, :n].double().sum()) - heads) <= 1e-5 * heads
        assert (w[s, n:] == 0).all()


def test_on_another_stream(cuda):
    """weigh_kv behind its inputs on a stream of the caller's, beside the current one's work."""
    c = Case(cuda, "paged", [900, 33, 64], 2, heads=128)
    want, got = torch.zeros_like(c.weights), torch.zeros_like(c.weights)
    c.run(want)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        c.run(got)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_long_rows_of_one_sequence(cuda):
    Case(cuda, "paged", [5000, 3], 1, heads=32, seed=4).check(AUTO)


def test_lengths_outside_their_regions(cuda):
    c = Case(cuda, "paged", [8, 40, 100, 30], 4)
    c.layout.kw["seq_lens"].copy_(torch.tensor([0, 40, 100, -3], dtype=torch.int32))
    start = c.weights.clone()
    c.rows[0] = c.rows[0][:0]
    c.rows[3] = c.rows[3][:0]
    for variant in (AUTO, PLAIN):
        c.run(kernel_variant=variant)
    got = (c.weights - start).cpu().view(-1)
    for s, w in enumerate(c.reference()[0]):
        at = weight_places(c.layout, s, len(w))
        assert ((got[at].double() - 2 * w).abs() <= 1e-5 * w + 1e-6).all()
    assert (got.view(4, -1)[0] == 0).all() and (got.view(4, -1)[3] == 0).all()


@pytest.mark.parametrize("variant", [AUTO, PLAIN])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_row_that_is_not_finite_stays_with_its_sequence(cuda, variant, bad):
    """Every token of the sequence sees row 7 (its weights are not numbers then); the others do not, nor do tokens before it."""
    c = Case(cuda, "paged", [50, 60, 70], 3)
    ref = c.reference()[0]
    data = [r.float().clone() for r in c.rows]
    data[1][59] = bad  # the newest row: only the last token sees it
    c.layout = Layout("paged", data, torch.bfloat16, cuda, block=64, seed=1)
    w = torch.zeros_like(c.weights)
    c.run(w, kernel_variant=variant)
    got = w.cpu().double().view(-1)
    for s in (0, 2):
        at = weight_places(c.layout, s, len(ref[s]))
        assert (got[at] - ref[s]).norm() <= 1e-5 * ref[s].norm()
    assert got[weight_places(c.layout, 1, 60)].isnan().all()


def test_same_bits_twice_and_captured(cuda):
    c, other = Case(cuda, "paged", [600, 90, 1500], 2, heads=32, seed=3), Case(cuda, "paged", [333, 64], 1, seed=4)
    outs = []
    for _ in range(3):
        w = torch.zeros_like(c.weights)
        c.run(w)
        outs.append(w)
    assert all(torch.equal(outs[0], w) for w in outs)
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    w, side0 = torch.zeros_like(c.weights), torch.zeros_like(other.weights)
    other.run(side0)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        c.run(w)
    for _ in range(3):
        w.zero_()
        graph.replay()
        side = torch.zeros_like(other.weights)
        other.run(side)
        torch.cuda.synchronize()
        assert torch.equal(w, outs[0]) and torch.equal(side, side0)
    c.layout.kw["seq_lens"].copy_(torch.tensor([100, 0, 1499], dtype=torch.int32))
    want = torch.zeros_like(w)
    c.run(want)
    w.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(w, want)


def test_refusals(cuda):
    c = Case(cuda, "paged", [40, 100], 3)
    cap = Case(cuda, "capacity", [40, 100], 3)
    off = Case(cuda, "packed", [40, 100], 3)
    for case, w in ((c, c.weights[:, :-1].contiguous()), (c, c.weights.double()), (c, c.weights.cpu()), (c, c.weights.t()),
                    (cap, cap.weights.view(-1)), (off, off.weights[:-1]), (off, off.weights.view(2, -1))):
        with pytest.raises(RuntimeError):
            case.run(w)
    with pytest.raises(RuntimeError, match="multiple of the batch"):
        F.weigh_kv(c.weights, c.layout.kv, c.q[:5, :, :128], c.q[:5, :, 128:], c.W_UK, c.cos, c.sin, c.cfg, **c.layout.kw)
    with pytest.raises(RuntimeError):
        c.run(kernel_variant=3)


def test_workspace_is_the_callers(cuda):
    lib = capi.load()
    c = Case(cuda, "capacity", [600, 90], 2, heads=16, q=torch.float32)
    want = torch.zeros_like(c.weights)
    c.run(want)
    q = c.q.contiguous()
    w = torch.zeros_like(want)
    a = capi.WeighArgs(kv_cache=c.layout.kv.data_ptr(), kv_dtype=capi.LA_DTYPE_BF16, total_rows=c.layout.kv.shape[0] * c.layout.kv.shape[1],
                       num_seqs=2, seq_len=c.layout.kv.shape[1], seq_lens=c.layout.kw["seq_lens"].data_ptr(), tokens_per_seq=2,
                       q_nope=q.data_ptr(), q_rope=q.data_ptr() + 512, q_dtype=capi.LA_DTYPE_F32, q_nope_token_stride=16 * 192,
                       q_nope_head_stride=192, q_rope_token_stride=16 * 192, q_rope_head_stride=192, rotate_q=1,
                       W_UK=c.W_UK.data_ptr(), w_uk_dtype=capi.LA_DTYPE_BF16, rope_cos=c.cos.data_ptr(), rope_sin=c.sin.data_ptr(),
                       rope_rows=c.cos.shape[0], weights=w.data_ptr(), cfg=capi.config(c.cfg))
    stream = torch.cuda.current_stream().cuda_stream
    for variant in (AUTO, PLAIN):
        a.kernel_variant = variant
        need = lib.la_weigh_kv_workspace_size(ctypes.byref(a))
        ws = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device=cuda)
        for base, size in ((ws.data_ptr() + 8, need), (None, 0)):
            a.workspace, a.workspace_bytes = base, size
            w.zero_()
            assert lib.la_weigh_kv(ctypes.byref(a), stream) == capi.LA_SUCCESS
            torch.cuda.synchronize()
            assert (w - want).norm() <= 1e-5 * want.norm()
        assert (ws[need + 8:] == 0xFF).all() and (ws[:8] == 0xFF).all()
