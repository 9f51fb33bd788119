"""GPU parity of functional.mla_decode_tree (la_mla_decode_tree) and functional.accept_kv (la_accept_kv) against the
64-bit references of tests/draft_cases.py: layouts, types, trees, sizes, rows that hold infinities or NaN, and a run
of the framework's calls as a speculating server makes them."""

from __future__ import annotations

import ctypes

import pytest
import torch

from conftest import assert_close
from draft_cases import ancestors, places, tree, tree_reference
from prompt_cases import Layout, as_double, tables, weights

from latent_attn import MLAConfig, capi
from latent_attn import functional as F

pytestmark = pytest.mark.gpu

AUTO, PLAIN, MFMA = 0, 1, 2


def config(heads, dc=512, dn=128, d_r=64, dv=128):
    return MLAConfig(5120, dc, dn, d_r, heads, dv)


class Case:
    def __init__(self, cuda, layout, rows, n, heads=16, kv=torch.bfloat16, q=torch.bfloat16, w=None, kind="random",
                 rotate_q=True, block=64, seed=1, dims=(512, 128, 64, 128), parents=None, data=None):
        dc, dn, d_r, dv = dims
        self.cfg, self.kv_type, self.q_type = config(heads, dc, dn, d_r, dv), kv, q
        g = torch.Generator().manual_seed(seed)
        data = data or [torch.randn(m, dc + d_r, generator=g).to(kv).float() for m in rows]
        self.layout = Layout(layout, data, kv, cuda, block=block, seed=seed)
        self.rows = [d.double() for d in data]
        self.q = torch.randn(len(rows) * n, heads, dn + d_r, generator=g).to(q).to(cuda)
        w = w or (kv if kv in (torch.float16, torch.bfloat16, torch.float32) else torch.bfloat16)
        self.W_UK, self.W_UV = (x.to(cuda) for x in weights(heads, w, seed + 1, dc, dn, dv))
        cos, sin = tables(max(rows), d_r)
        self.cos, self.sin = cos.to(cuda), sin.to(cuda)
        self.parents = parents or [tree(n, seed + s, kind) for s in range(len(rows))]
        self.par = torch.tensor(self.parents, dtype=torch.int32, device=cuda)
        self.rotate_q, self.dn, self.n = rotate_q, dn, n

    def run(self, **kw):
        kw = {**self.layout.kw, "rotate_q": self.rotate_q, **kw}
        return F.mla_decode_tree(self.layout.kv, self.q[..., :self.dn], self.q[..., self.dn:], self.W_UK, self.W_UV,
                                 self.cos, self.sin, self.cfg, self.par, **kw)

    def reference(self):
        q = as_double(self.q)
        return tree_reference(self.rows, q[..., :self.dn], q[..., self.dn:], as_double(self.W_UK), as_double(self.W_UV),
                              as_double(self.cos), as_double(self.sin), self.parents, self.rotate_q)

    def check(self, got, plain, what=""):
        ref = self.reference()
        kind = "f32" if plain and got.dtype == torch.float32 else "bf16"
        assert_close(got.double().cpu().numpy(), ref.numpy(), kind, what)


@pytest.mark.parametrize("layout", ["uniform", "capacity", "packed", "packed_capacity", "paged"])
@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn])
def test_plain_by_layout_and_type(cuda, layout, kv):
    rows = [70] * 3 if layout == "uniform" else [9, 70, 131]
    c = Case(cuda, layout, rows, 9, heads=3, kv=kv, q=torch.float32, block=16)
    c.check(c.run(kernel_variant=PLAIN), True, f"{layout} {kv}")


@pytest.mark.parametrize("n,kind", [(1, "star"), (2, "star"), (2, "chain"), (31, "random"), (32, "chain"), (33, "random"),
                                    (63, "star"), (64, "chain"), (64, "random")])
@pytest.mark.parametrize("variant", [AUTO, PLAIN])
def test_trees(cuda, n, kind, variant):
    """Contexts of no row, one, and around the tiles' borders, trees that end in and on them."""
    rows = [n, n + 1, n + 31, n + 32, n + 33, 150 + n]
    c = Case(cuda, "paged", rows, n, heads=16, kind=kind, seed=n)
    c.check(c.run(kernel_variant=variant), variant == PLAIN, f"{n} {kind}")


@pytest.mark.parametrize("q", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rotate_q", [False, True])
@pytest.mark.parametrize("variant", [AUTO, PLAIN])
def test_queries_and_outputs(cuda, q, rotate_q, variant):
    c = Case(cuda, "capacity", [40, 100], 7, q=q, rotate_q=rotate_q)
    for out in (None, torch.float32, torch.float16, torch.bfloat16):
        got = c.run(kernel_variant=variant, out_dtype=out)
        assert got.dtype == (out or q)
        c.check(got, variant == PLAIN, f"{q} {rotate_q} {out}")


def test_packed_queries_are_taken_where_they_lie(cuda):
    c = Case(cuda, "capacity", [40, 100], 7, q=torch.float32, rotate_q=False)
    nope, rope = c.q[..., :128].contiguous(), c.q[..., 128:].contiguous()
    before = nope.clone(), rope.clone()
    got = F.mla_decode_tree(c.layout.kv, nope, rope, c.W_UK, c.W_UV, c.cos, c.sin, c.cfg, c.par, **c.layout.kw)
    c.check(got, False)
    assert torch.equal(nope, before[0]) and torch.equal(rope, before[1])


@pytest.mark.parametrize("dims,heads", [((64, 32, 16, 24), 5), ((512, 128, 64, 128), 3), ((96, 40, 6, 33), 2), ((1024, 64, 128, 64), 1)])
def test_other_head_shapes(cuda, dims, heads):
    c = Case(cuda, "packed_capacity", [5, 60, 77], 5, heads=heads, kv=torch.float32, q=torch.float32, dims=dims)
    c.check(c.run(), True, str(dims))


# 64 nodes x 128 heads leave a chip of 256 compute units four chunks: several
# sequences in one, a sequence over several, none in a sequence without rows, and, with
# sequences of about one length, a chunk each
@pytest.mark.parametrize("layout", ["capacity", "packed_capacity", "packed", "paged"])
@pytest.mark.parametrize("rows", [[70, 900, 64, 65, 300, 96, 128], [1200], [64, 64, 64, 64], [63, 700, 1, 690, 64, 10],
                                  [10, 20, 300]])
def test_chunks_across_sequences(cuda, layout, rows):
    case = Case(cuda, layout, rows, 64, heads=128, seed=len(rows))
    case.check(case.run(), False, (layout, rows))


@pytest.mark.parametrize("rows,n,heads", [([40, 100], 7, 16), ([700, 64, 130], 64, 128)])
@pytest.mark.parametrize("w", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float16])
def test_weights_and_outputs_of_every_type(cuda, rows, n, heads, w, kv):
    c = Case(cuda, "capacity", rows, n, heads=heads, kv=kv, w=w)
    ref = c.reference().numpy()
    for out in (torch.float32, torch.float16, torch.bfloat16):
        got = c.run(kernel_variant=MFMA, out_dtype=out)
        assert got.dtype == out
        assert_close(got.double().cpu().numpy(), ref, "bf16", f"{w} {out}")


@pytest.mark.parametrize("dims", [(512, 64, 64, 128), (512, 128, 64, 96), (512, 48, 64, 40), (512, 192, 64, 128)])
@pytest.mark.parametrize("rows,n,heads", [([40, 100], 7, 16), ([500, 64], 32, 64)])
def test_other_heads_over_the_same_rows(cuda, dims, rows, n, heads):
    """The matrix cores' attention with absorption and projection of other widths."""
    c = Case(cuda, "paged", rows, n, heads=heads, dims=dims)
    c.check(c.run(kernel_variant=MFMA), False, dims)


def test_an_output_out_of_line(cuda):
    """An output that is not aligned to 16 bytes, and nothing written beside it."""
    lib = capi.load()
    c = Case(cuda, "capacity", [700, 64, 130], 64, heads=128)
    want = c.run(out_dtype=torch.bfloat16)
    room = torch.full((want.numel() + 64,), 7.0, dtype=torch.bfloat16, device=cuda)
    kv = c.layout.kv
    a = capi.TreeArgs(kv_cache=kv.data_ptr(), kv_dtype=capi.LA_DTYPE_BF16, total_rows=kv.shape[0] * kv.shape[1], num_seqs=3,
                      seq_len=kv.shape[1], seq_lens=c.layout.kw["seq_lens"].data_ptr(), nodes=64, parents=c.par.data_ptr(),
                      q_nope=c.q.data_ptr(), q_rope=c.q.data_ptr() + 2 * 128, q_dtype=capi.LA_DTYPE_BF16,
                      q_nope_token_stride=128 * 192, q_nope_head_stride=192, q_rope_token_stride=128 * 192,
                      q_rope_head_stride=192, rotate_q=1, W_UK=c.W_UK.data_ptr(), w_uk_dtype=capi.LA_DTYPE_BF16,
                      W_UV=c.W_UV.data_ptr(), w_uv_dtype=capi.LA_DTYPE_BF16, rope_cos=c.cos.data_ptr(),
                      rope_sin=c.sin.data_ptr(), rope_rows=c.cos.shape[0], output=room.data_ptr() + 2 * 3,
                      out_dtype=capi.LA_DTYPE_BF16, cfg=capi.config(c.cfg))
    assert lib.la_mla_decode_tree(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == capi.LA_SUCCESS
    torch.cuda.synchronize()
    got = room[3:3 + want.numel()].view_as(want)
    assert_close(got.double().cpu().numpy(), want.double().cpu().numpy(), "bf16")
    assert (room[:3] == 7).all() and (room[3 + want.numel():] == 7).all()


def test_captured_with_many_heads(cuda):
    """The chunks follow the lengths at every replay: of one long sequence, of equal ones, of none."""
    c = Case(cuda, "paged", [900, 800, 700, 64], 64, heads=128)
    par0, lens = c.par.clone(), c.layout.kw["seq_lens"]
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    c.run()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        got = c.run()
    for rows in ([900, 800, 700, 64], [900, 0, 0, 0], [100, 100, 100, 64], [0, 0, 0, 0], [70, 800, 63, 64], [900, 800, 700, 64]):
        lens.copy_(torch.tensor(rows, dtype=torch.int32))
        graph.replay()
        eager = c.run()
        torch.cuda.synchronize()
        assert torch.equal(got.view(torch.int16), eager.view(torch.int16)), rows
        short = torch.tensor([n < 64 for n in rows], device=cuda).repeat_interleave(64)
        assert (got[short] == 0).all() and got.isfinite().all()
    c.check(got, False)
    assert torch.equal(c.par, par0)


@pytest.mark.parametrize("count,n,heads", [(150, 3, 16), (70, 16, 64), (65, 1, 16), (300, 2, 16), (600, 8, 16)])
def test_more_sequences_than_lanes(cuda, count, n, heads):
    rows = [(37 * i * i + 11 * i) % 190 for i in range(count)]
    case = Case(cuda, "capacity", rows, n, heads=heads)
    case.check(case.run(), False, (count, n, heads))


@pytest.mark.parametrize("block", [7, 16, 48, 96])
def test_block_sizes(cuda, block):
    """A tile of 32 rows lies in one block, or the plain kernel runs."""
    case = Case(cuda, "paged", [200, 20, 97], 9, block=block)
    case.check(case.run(), False, block)


@pytest.mark.parametrize("variant", [AUTO, PLAIN])
@pytest.mark.parametrize("q", [torch.float32, torch.bfloat16])
def test_queries_out_of_line(cuda, variant, q):
    """Views whose elements are not aligned to whole vectors, by token, head or address."""
    for pad, skip in ((1, 0), (4, 1), (3, 2)):
        c = Case(cuda, "capacity", [150, 64, 300], 6, q=q, seed=pad)
        wide = torch.zeros(*c.q.shape[:2], c.q.shape[2] + pad, dtype=q, device=cuda)
        wide[..., skip:skip + c.q.shape[2]] = c.q
        c.q = wide[..., skip:skip + c.q.shape[2]]
        c.check(c.run(kernel_variant=variant, out_dtype=torch.float32), variant == PLAIN, (pad, skip))


def test_parents_outside_their_range_are_none(cuda):
    parents = [[5, -7, 0, 3, 2 ** 30, 1, 4], [-1, 0, 1, -2 ** 31, 3, 6, 5]]
    c = Case(cuda, "paged", [50, 90], 7, parents=parents)
    clean = [[p if 0 <= p < j else -1 for j, p in enumerate(t)] for t in parents]
    c.parents = clean
    for variant in (AUTO, PLAIN):
        c.check(c.run(kernel_variant=variant), variant == PLAIN)


def test_sequences_without_a_tree(cuda):
    """Empty slots of a padded batch, sequences shorter than their trees, and lengths outside their regions."""
    c = Case(cuda, "paged", [8, 40, 100, 30], 8)
    lens = c.layout.kw["seq_lens"]
    want = c.reference()
    lens.copy_(torch.tensor([0, 7, 100, -3], dtype=torch.int32))
    want[:16] = 0
    want[24:] = 0
    for variant in (AUTO, PLAIN):
        got = c.run(kernel_variant=variant, out_dtype=torch.float32)
        assert_close(got.cpu().numpy(), want.numpy(), "bf16")
        assert (got[:16] == 0).all() and (got[24:] == 0).all()


@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.float32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("part", ["latent", "rope"])
@pytest.mark.parametrize("variant", [AUTO, PLAIN])
def test_rows_that_are_not_finite_reach_only_those_that_see_them(cuda, kv, bad, part, variant):
    if kv == torch.float8_e4m3fn and bad == bad:
        pytest.skip("E4M3 has no infinity")
    n = 12
    for L, node in ((40, 5), (40, 11), (96, 0), (n, 3)):
        g = torch.Generator().manual_seed(L + node)
        data = [torch.randn(L, 576, generator=g).to(kv).float()]
        c = Case(cuda, "paged", [L], n, kv=kv, data=data, seed=node)
        clean = c.reference()
        data[0][L - n + node, 100 if part == "latent" else 530] = bad
        c.layout = Layout("paged", data, kv, cuda, block=64, seed=node)
        got = c.run(kernel_variant=variant, out_dtype=torch.float32).double().cpu()
        sees = torch.tensor([node in a for a in ancestors(c.parents[0])])
        assert sees.any() and not sees.all()
        assert_close(got[~sees].numpy(), clean[~sees].numpy(), "bf16")
        if bad != bad or part == "latent":
            assert got[sees].isnan().all()


# 64 nodes x 128 heads: the kernel of 128 heads per workgroup (fewer take the one of 16)
@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("bad,part", [(float("nan"), "latent"), (float("inf"), "latent"), (float("nan"), "rope")])
def test_rows_that_are_not_finite_with_many_heads(cuda, kv, bad, part):
    if kv == torch.float8_e4m3fn and bad == bad:
        pytest.skip("e4m3 has no infinities")
    n = 64
    for L, node in ((150, 5), (224, 11), (700, 63)):
        g = torch.Generator().manual_seed(L + node)
        data = [torch.randn(L, 576, generator=g).to(kv).float()]
        c = Case(cuda, "paged", [L], n, heads=128, kv=kv, data=data, seed=node)
        clean = c.reference()
        data[0][L - n + node, 100 if part == "latent" else 530] = bad
        c.layout = Layout("paged", data, kv, cuda, block=64, seed=node)
        got = c.run(kernel_variant=MFMA, out_dtype=torch.float32).double().cpu()
        sees = torch.tensor([node in a for a in ancestors(c.parents[0])])
        assert sees.any() and not sees.all()
        assert_close(got[~sees].numpy(), clean[~sees].numpy(), "bf16")
        assert got[sees].isnan().all()


# the 16-head kernel's largest launches and the 128-head kernel's smallest: 512 (under 128 heads to a sequence: 1024)
# rows per 16 heads and compute unit, of 256
@pytest.mark.parametrize("rows,n,heads", [([8000, 40], 1, 128), ([4700, 40, 700], 3, 128), ([36000], 7, 16), ([38000], 7, 16),
                                          ([9000, 300, 129], 1, 16)])
@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float8_e4m3fn])
def test_around_the_smaller_kernels_range(cuda, rows, n, heads, kv):
    case = Case(cuda, "packed_capacity", rows, n, heads=heads, kv=kv)
    case.check(case.run(), False, (rows, n, heads))


def test_scores_far_apart(cuda):
    """Rows scaled so that scores jump by hundreds between context and nodes, either way."""
    for scale in (6.0, 1 / 6.0):
        g = torch.Generator().manual_seed(3)
        data = [torch.cat([torch.randn(130, 576, generator=g) * scale, torch.randn(20, 576, generator=g) / scale]).bfloat16().float()]
        c = Case(cuda, "capacity", [150], 20, data=data, q=torch.float32)
        ref = c.reference()
        got = c.run(kernel_variant=PLAIN).double().cpu()
        assert (got - ref).norm() <= 1e-5 * ref.norm()
        got = c.run(kernel_variant=AUTO).double().cpu()
        assert got.isfinite().all() and (got - ref).norm() <= 4e-2 * ref.norm()


def test_refusals(cuda):
    c = Case(cuda, "capacity", [40, 100], 7)
    args = [c.layout.kv, c.q[..., :128], c.q[..., 128:], c.W_UK, c.W_UV, c.cos, c.sin, c.cfg, c.par]
    kw = dict(c.layout.kw)

    def refused(match, *, at=None, value=None, **more):
        a = list(args)
        if at is not None:
            a[at] = value
        with pytest.raises((RuntimeError, ValueError), match=match):
            F.mla_decode_tree(*a, **{**kw, **more})

    refused("q_rope must be", at=1, value=c.q[:13, :, :128])
    refused("parents", at=8, value=c.par[:, :6].contiguous())
    refused("parents", at=8, value=c.par.long())
    refused("parents", at=8, value=c.par.cpu())
    refused("same dtype", at=2, value=c.q[..., 128:].float())
    refused("last dimension", at=1, value=torch.zeros(14, 16, 256, device=cuda, dtype=torch.bfloat16)[..., ::2])
    refused("W_UK shape", at=3, value=c.W_UK[:-1])
    big = torch.zeros(2 * 65, 16, 192, device=cuda)
    with pytest.raises(RuntimeError, match="nodes"):
        F.mla_decode_tree(c.layout.kv, big[..., :128], big[..., 128:], *args[3:8],
                          torch.zeros(2, 65, dtype=torch.int32, device=cuda), **kw)


# ---- accepted paths ---------------------------------------------------------------------------------------------------


def accept_reference(rows, n, path):
    """(rows that stay, their number) of one sequence."""
    L = rows.shape[0]
    if L < n:
        return rows
    keep, last = [], -1
    for p in path:
        if not last < p < n:
            break
        keep.append(L - n + p)
        last = p
    return torch.cat([rows[:L - n], rows[keep]])


@pytest.mark.parametrize("layout", ["capacity", "packed_capacity", "paged"])
@pytest.mark.parametrize("kv,dims", [(torch.bfloat16, (512, 64)), (torch.float32, (512, 64)), (torch.float8_e4m3fn, (512, 64)),
                                     (torch.float16, (33, 6)), (torch.float8_e4m3fn, (33, 6)), (torch.float16, (1024, 256)),
                                     (torch.float32, (2048, 64))])
def test_accept(cuda, layout, kv, dims):
    width, n = sum(dims), 64
    g = torch.Generator().manual_seed(5)
    rows = [100, 64, 63, 200, 65, 70, 90, 64]
    paths = [[0, 3, 17, 63], list(range(64)), [0, 1, 2], [63], [], [0, 1, 2, 2, 5], [5, 64, 7], [1, 2, 3] + list(range(5, 64))]
    data = [torch.randn(m, width, generator=g).to(kv).float() for m in rows]
    lay = Layout(layout, data, kv, cuda, block=16, junk=0.0)
    lens = lay.kw["seq_lens"]
    before = lay.kv.clone()
    path = torch.tensor([(p + [-1] * n)[:n] for p in paths], dtype=torch.int32, device=cuda)
    kw = {k: v for k, v in lay.kw.items() if k != "seq_lens"}
    F.accept_kv(lay.kv, lens, n, path, MLAConfig(5120, dims[0], 128, dims[1], 16, 128), **kw)
    flat, old = (x.view(torch.uint8).view(-1, width * lay.kv.element_size()).cpu() for x in (lay.kv, before))
    touched = torch.zeros(flat.shape[0], dtype=torch.bool)
    for s, d in enumerate(data):
        want = accept_reference(torch.arange(rows[s])[:, None], n, paths[s])[:, 0]
        assert int(lens[s]) == len(want), s
        at = places(lay, s, rows[s])
        assert torch.equal(flat[at[:len(want)]], old[at[want]]), s
        touched[at[:len(want)]] = True
    assert torch.equal(flat[~touched], old[~touched])  # nothing else has changed


def test_accept_leaves_bad_lengths_alone(cuda):
    kv = torch.randn(3, 32, 576, device=cuda).bfloat16()
    before = kv.clone()
    lens = torch.tensor([33, -1, 3], dtype=torch.int32, device=cuda)
    F.accept_kv(kv, lens, 4, torch.tensor([[1, 2, 3, -1]] * 3, dtype=torch.int32, device=cuda), MLAConfig.deepseek_v2())
    assert lens.tolist() == [33, -1, 3] and torch.equal(kv, before)


def test_accept_refusals(cuda):
    kv = torch.zeros(2, 32, 576, device=cuda).bfloat16()
    lens, cfg = torch.zeros(2, dtype=torch.int32, device=cuda), MLAConfig.deepseek_v2()
    path = torch.zeros(2, 4, dtype=torch.int32, device=cuda)
    for bad in (lambda: F.accept_kv(kv, lens, 5, path, cfg), lambda: F.accept_kv(kv, lens.long(), 4, path, cfg),
                lambda: F.accept_kv(kv, lens[:1], 4, path, cfg), lambda: F.accept_kv(kv, lens, 0, path[:, :0], cfg),
                lambda: F.accept_kv(kv, lens, 65, torch.zeros(2, 65, dtype=torch.int32, device=cuda), cfg),
                lambda: F.accept_kv(kv[..., :500].contiguous(), lens, 4, path, cfg),
                lambda: F.accept_kv(kv, lens, 4, path.cpu(), cfg)):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.parametrize("block", [0, 64])
def test_a_speculating_run(cuda, block):
    """Append a tree, attend it, keep a path, append the next: every path's tokens get what a chain of them gets."""
    heads, B, n, cap = 16, 3, 10, 256
    cfg = config(heads)
    g = torch.Generator().manual_seed(9)
    W_UK, W_UV = (x.to(cuda) for x in weights(heads, torch.bfloat16, 2))
    cos, sin = (x.to(cuda) for x in tables(cap))
    kw = {}
    if block:
        table = torch.randperm(B * cap // block, generator=g).int().view(B, -1).to(cuda)
        kw = {"block_table": table, "block_size": block}
        kv = torch.zeros(B * cap, 576, dtype=torch.bfloat16, device=cuda)
    else:
        kv = torch.zeros(B, cap, 576, dtype=torch.bfloat16, device=cuda)
    lens = torch.zeros(B, dtype=torch.int32, device=cuda)

    def rand(*shape):
        return torch.randn(*shape, generator=g).bfloat16().to(cuda)

    F.append_kv(kv, lens, rand(B, 50, 512), rand(B, 50, 64), cfg, **kw)
    kept = None
    for step in range(3):
        parents = [tree(n, 10 * step + s) for s in range(B)]
        paths = []
        for s, p in enumerate(parents):
            path, j = [], n - 1 - s
            while j >= 0:
                path.insert(0, j)
                j = p[j]
            paths.append(path)
        c_t, k_r, q = rand(B, n, 512), rand(B, n, 64), rand(B * n, heads, 192)
        before = lens.tolist()
        F.append_kv(kv, lens, c_t, k_r, cfg, **kw)
        got = F.mla_decode_tree(kv, q[..., :128], q[..., 128:], W_UK, W_UV, cos, sin, cfg,
                                torch.tensor(parents, dtype=torch.int32, device=cuda), seq_lens=lens, rotate_q=True, **kw)
        F.accept_kv(kv, lens, n, torch.tensor([(p + [-1] * n)[:n] for p in paths], dtype=torch.int32, device=cuda), cfg, **kw)
        assert lens.tolist() == [b + len(p) for b, p in zip(before, paths)]
        # the accepted tokens as a piece of a prompt, over the rows that stayed
        at = torch.tensor([s * n + j for s, p in enumerate(paths) for j in p], device=cuda)
        offs = torch.tensor([0] + [sum(len(p) for p in paths[:s + 1]) for s in range(B)], dtype=torch.int32, device=cuda)
        chain = F.mla_prefill(kv, q[at][..., :128], q[at][..., 128:], W_UK, W_UV, cos, sin, cfg, q_offsets=offs,
                              seq_lens=lens, rotate_q=True, **kw)
        assert_close(got[at].double().cpu().numpy(), chain.double().cpu().numpy(), "bf16", f"step {step}")
        kept = got
    assert kept is not None


def test_two_streams_and_capture(cuda):
    """A captured tree step and acceptance, replayed over other lengths, rows and trees, beside an eager one."""
    c, other = Case(cuda, "paged", [60, 90, 10], 8, seed=3), Case(cuda, "paged", [33, 64, 120], 8, seed=4)
    want, want2 = c.run(), other.run()
    lens0 = c.layout.kw["seq_lens"].clone()
    path = torch.tensor([[0, 2, 5] + [-1] * 5] * 3, dtype=torch.int32, device=cuda)
    kw = {k: v for k, v in c.layout.kw.items() if k != "seq_lens"}
    kv0 = c.layout.kv.clone()
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        got = c.run()
        F.accept_kv(c.layout.kv, c.layout.kw["seq_lens"], 8, path, c.cfg, **kw)
    for i in range(3):
        c.layout.kv.copy_(kv0)
        c.layout.kw["seq_lens"].copy_(lens0)
        graph.replay()
        side = other.run()
        torch.cuda.synchronize()
        assert torch.equal(got.view(torch.int16), want.view(torch.int16)), i
        assert torch.equal(side.view(torch.int16), want2.view(torch.int16)), i
        assert c.layout.kw["seq_lens"].tolist() == [n - 5 for n in lens0.tolist()]
    c.layout.kw["seq_lens"].copy_(torch.tensor([20, 0, 9], dtype=torch.int32))
    c.par.fill_(-1)
    c.layout.kv.copy_(kv0)
    eager = c.run()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got.view(torch.int16), eager.view(torch.int16))


def test_workspace_is_the_callers(cuda):
    """The C entry with a workspace of exactly its size, at an odd address, and with none."""
    lib = capi.load()
    c = Case(cuda, "capacity", [60, 90], 8, q=torch.float32)
    want = c.run()
    q = c.q.contiguous()
    out = torch.empty_like(want)
    a = capi.TreeArgs(kv_cache=c.layout.kv.data_ptr(), kv_dtype=capi.LA_DTYPE_BF16, total_rows=c.layout.kv.shape[0] * c.layout.kv.shape[1],
                      num_seqs=2, seq_len=c.layout.kv.shape[1], seq_lens=c.layout.kw["seq_lens"].data_ptr(), nodes=8,
                      parents=c.par.data_ptr(), q_nope=q.data_ptr(), q_rope=q.data_ptr() + 512, q_dtype=capi.LA_DTYPE_F32,
                      q_nope_token_stride=16 * 192, q_nope_head_stride=192, q_rope_token_stride=16 * 192, q_rope_head_stride=192,
                      rotate_q=1, W_UK=c.W_UK.data_ptr(), w_uk_dtype=capi.LA_DTYPE_BF16, W_UV=c.W_UV.data_ptr(),
                      w_uv_dtype=capi.LA_DTYPE_BF16, rope_cos=c.cos.data_ptr(), rope_sin=c.sin.data_ptr(),
                      rope_rows=c.cos.shape[0], output=out.data_ptr(), out_dtype=capi.LA_DTYPE_F32, cfg=capi.config(c.cfg))
    stream = torch.cuda.current_stream().cuda_stream
    for variant in (AUTO, PLAIN):
        a.kernel_variant = variant
        need = lib.la_mla_decode_tree_workspace_size(ctypes.byref(a))
        ws = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device=cuda)
        for base, size in ((ws.data_ptr() + 8, need), (None, 0)):
            a.workspace, a.workspace_bytes = base, size
            out.fill_(float("nan"))
            assert lib.la_mla_decode_tree(ctypes.byref(a), stream) == capi.LA_SUCCESS
            torch.cuda.synchronize()
            assert_close(out.cpu().numpy(), want.cpu().numpy(), "bf16")
        assert (ws[need + 8:] == 0xFF).all() and (ws[:8] == 0xFF).all()
