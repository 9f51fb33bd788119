"""GPU tests of functional.evict_kv (la_evict_kv): what stays, where it goes, what is left alone, and its use with
weigh_kv and the decode step. Rows and positions are moved, not computed: everything is compared exactly."""

from __future__ import annotations

import ctypes

import pytest
import torch

from draft_cases import evict_reference, places, room, weight_places
from prompt_cases import Layout, tables, weights

from latent_attn import MLAConfig, capi
from latent_attn import functional as F

pytestmark = pytest.mark.gpu


def check(cuda, layout, rows, keep, first, last, kv=torch.bfloat16, dims=(512, 64), block=64, seed=1, w=None, passes=1):
    width = sum(dims)
    g = torch.Generator().manual_seed(seed)
    data = [torch.randn(m, width, generator=g).to(kv).float() for m in rows]
    lay = Layout(layout, data, kv, cuda, block=block, junk=0.0, seed=seed)
    lens = lay.kw["seq_lens"]
    cfg = MLAConfig(5120, dims[0], 128, dims[1], 16, 128)
    wts = torch.rand(*room(lay), generator=g)
    if w is not None:
        for s in range(len(rows)):
            wts.view(-1)[weight_places(lay, s, rows[s])] = w(s, rows[s], g)
    wts = wts.to(cuda)
    kw = {k: v for k, v in lay.kw.items() if k != "seq_lens"}
    old, w0 = lay.kv.clone(), wts.clone()
    kept = F.evict_kv(lay.kv, lens, wts, cfg, keep, first=first, last=last, **kw).cpu()
    assert kept.shape == (len(rows), keep) and kept.dtype == torch.int32
    flat, was = (x.view(torch.uint8).view(-1, width * lay.kv.element_size()).cpu() for x in (lay.kv, old))
    wts, w0 = wts.cpu().view(-1), w0.cpu().view(-1)
    touched, weighed = torch.zeros(flat.shape[0], dtype=torch.bool), torch.zeros(wts.numel(), dtype=torch.bool)
    for s, L in enumerate(rows):
        at, wat = places(lay, s, L), weight_places(lay, s, L)
        want = torch.tensor(evict_reference(w0[wat].tolist(), keep, first, last), dtype=torch.long)
        m = len(want)
        assert int(lens[s]) == m, s
        assert kept[s, :m].tolist() == want.tolist() and (kept[s, m:] == -1).all(), s
        assert torch.equal(flat[at[:m]], was[at[want]]), s
        assert torch.equal(wts[wat[:m]].view(torch.int32), w0[wat[want]].view(torch.int32)), s
        assert (wts[wat[m:]] == 0).all(), s
        touched[at[:m]] = True
        weighed[wat] = True
    assert torch.equal(flat[~touched], was[~touched])
    assert torch.equal(wts[~weighed], w0[~weighed])


ROWS = [1, 40, 63, 64, 65, 100, 257, 1000]


@pytest.mark.parametrize("layout", ["capacity", "packed_capacity", "paged"])
@pytest.mark.parametrize("keep,first,last", [(64, 4, 16), (64, 0, 0), (64, 64, 0), (64, 0, 64), (64, 20, 44), (1, 0, 0),
                                             (1, 0, 1), (0, 0, 0), (255, 1, 1), (2000, 4, 16)])
def test_what_stays(cuda, layout, keep, first, last):
    check(cuda, layout, ROWS, keep, first, last)


@pytest.mark.parametrize("kv,dims", [(torch.float32, (512, 64)), (torch.float16, (512, 64)), (torch.float8_e4m3fn, (512, 64)),
                                     (torch.float16, (33, 6)), (torch.float8_e4m3fn, (33, 6)), (torch.bfloat16, (1024, 256)),
                                     (torch.float32, (3, 2)), (torch.float16, (34, 4)), (torch.float16, (36, 6))])
def test_types_and_row_sizes(cuda, kv, dims):
    check(cuda, "paged", [300, 17, 129], 50, 3, 7, kv=kv, dims=dims, block=16)
    check(cuda, "packed_capacity", [300, 17, 129], 50, 3, 7, kv=kv, dims=dims)


def test_long_sequences(cuda):
    check(cuda, "capacity", [5000, 4096, 4097, 1024, 1025, 9000], 1000, 4, 100, dims=(48, 16))
    check(cuda, "paged", [40000, 70000], 33000, 0, 1, dims=(6, 2), block=128)


@pytest.mark.parametrize("name", ["equal", "two", "zeros", "signs", "nan", "infinite", "low bits", "rising", "falling", "all nan"])
def test_weights_that_are_hard_to_rank(cuda, name):
    def w(s, n, g):
        if name == "equal":
            return torch.full((n,), 0.25)
        if name == "two":
            return torch.randint(0, 2, (n,), generator=g).float()
        if name == "zeros":
            return torch.where(torch.rand(n, generator=g) < 0.5, 0.0, -0.0)
        if name == "signs":
            return torch.randn(n, generator=g)
        if name == "rising":
            return torch.arange(n).float()
        if name == "falling":
            return -torch.arange(n).float()
        if name == "low bits":  # keys that differ in their last bits alone
            return (torch.randint(0, 5, (n,), generator=g) + 0x3F800000).int().view(torch.float32)
        x = torch.randn(n, generator=g)
        r = torch.rand(n, generator=g)
        if name == "nan":
            return torch.where(r < 0.7, float("nan"), x)
        if name == "all nan":
            return torch.full((n,), float("nan"))
        return torch.where(r < 0.3, float("inf"), torch.where(r < 0.6, -float("inf"), x))

    check(cuda, "paged", [1, 70, 300, 1500, 2049], 60, 2, 5, w=w, dims=(6, 2))


def test_lengths_outside_their_regions(cuda):
    kv = torch.randn(3, 64, 576, device=cuda).bfloat16()
    before = kv.clone()
    wts = torch.arange(192, dtype=torch.float32, device=cuda).view(3, 64)
    lens = torch.tensor([-5, 1000, 10], dtype=torch.int32, device=cuda)
    kept = F.evict_kv(kv, lens, wts, MLAConfig.deepseek_v2(), 16)
    # a length past its region counts as the region
    assert lens.tolist()[1:] == [16, 10] and kept[1].tolist() == list(range(48, 64))
    assert (kept[0] == -1).all() and torch.equal(kv[0], before[0]) and torch.equal(kv[2], before[2])


def test_refusals(cuda):
    cfg = MLAConfig.deepseek_v2()
    kv, lens = torch.zeros(2, 32, 576, device=cuda).bfloat16(), torch.zeros(2, dtype=torch.int32, device=cuda)
    w = torch.zeros(2, 32, device=cuda)
    for bad in (lambda: F.evict_kv(kv, lens, w, cfg, 8, first=5, last=4), lambda: F.evict_kv(kv, lens, w, cfg, -1),
                lambda: F.evict_kv(kv, lens, w, cfg, 8, first=-1), lambda: F.evict_kv(kv, lens, w, cfg, 8, last=-1),
                lambda: F.evict_kv(kv, lens, w[:, :31].contiguous(), cfg, 8), lambda: F.evict_kv(kv, lens, w.half(), cfg, 8),
                lambda: F.evict_kv(kv, lens.long(), w, cfg, 8), lambda: F.evict_kv(kv, lens.cpu(), w, cfg, 8),
                lambda: F.evict_kv(kv, lens[:1], w, cfg, 8), lambda: F.evict_kv(kv.view(64, 576), lens, w, cfg, 8),
                lambda: F.evict_kv(kv, lens, w, cfg, 1 << 31)):
        with pytest.raises((RuntimeError, TypeError)):
            bad()


def test_without_sequences_or_rows(cuda):
    cfg = MLAConfig.deepseek_v2()
    kept = F.evict_kv(torch.zeros(0, 32, 576, device=cuda), torch.zeros(0, dtype=torch.int32, device=cuda),
                      torch.zeros(0, 32, device=cuda), cfg, 8)
    assert kept.shape == (0, 8)
    kept = F.evict_kv(torch.zeros(2, 0, 576, device=cuda), torch.zeros(2, dtype=torch.int32, device=cuda),
                      torch.zeros(2, 0, device=cuda), cfg, 8)
    assert kept.tolist() == [[-1] * 8] * 2


@pytest.mark.parametrize("block", [0, 64])
def test_a_run_under_a_budget(cuda, block):
    """Append, weigh, decode, evict in turn: what the cache holds is what a cache of the kept rows alone holds."""
    heads, B, cap, keep = 16, 3, 192, 100
    cfg = MLAConfig(5120, 512, 128, 64, heads, 128)
    g = torch.Generator().manual_seed(2)
    W_UK, W_UV = (x.to(cuda) for x in weights(heads, torch.bfloat16, 2))
    cos, sin = (x.to(cuda) for x in tables(cap))
    kw = {}
    if block:
        kw = {"block_table": torch.randperm(B * cap // block, generator=g).int().view(B, -1).to(cuda), "block_size": block}
        kv = torch.zeros(B * cap, 576, dtype=torch.bfloat16, device=cuda)
    else:
        kv = torch.zeros(B, cap, 576, dtype=torch.bfloat16, device=cuda)
    lens = torch.zeros(B, dtype=torch.int32, device=cuda)
    wts = torch.zeros(B, cap, device=cuda)
    mirror = torch.zeros(B, 0, 576, dtype=torch.bfloat16, device=cuda)
    for step in range(4):
        new = torch.randn(B, 60 if step == 0 else 40, 576, generator=g).bfloat16().to(cuda)
        F.append_kv(kv, lens, new[..., :512].contiguous(), new[..., 512:].contiguous(), cfg, **kw)
        mirror = torch.cat([mirror, new], 1)
        q = torch.randn(B, heads, 192, generator=g).to(cuda)
        args = (q[..., :128].contiguous(), q[..., 128:].contiguous(), W_UK)
        F.weigh_kv(wts, kv, *args, cos, sin, cfg, seq_lens=lens, **kw)
        alone = torch.zeros(B, mirror.shape[1], device=cuda)
        F.weigh_kv(alone, mirror, *args, cos, sin, cfg)
        assert torch.allclose(wts.sum(1), torch.full((B,), float(heads * (step + 1)), device=cuda), rtol=0.5)
        kept = F.evict_kv(kv, lens, wts, cfg, keep, first=4, last=20, **kw)
        if mirror.shape[1] > keep:
            mirror = mirror.gather(1, kept.long()[..., None].expand(-1, -1, 576))
        assert lens.tolist() == [mirror.shape[1]] * B
        out = F.mla_decode(kv, *args, W_UV, cos, sin, cfg, seq_lens=lens, **kw)
        want = F.mla_decode(mirror.contiguous(), *args, W_UV, cos, sin, cfg)
        assert (out - want).norm() <= 1e-2 * want.norm()


def test_captured(cuda):
    g = torch.Generator().manual_seed(2)
    cfg = MLAConfig.deepseek_v2()
    kv0 = torch.randn(4, 700, 576, generator=g).bfloat16().to(cuda)
    w0 = torch.rand(4, 700, generator=g).to(cuda)
    l0 = torch.tensor([700, 0, 300, 699], dtype=torch.int32, device=cuda)

    def fresh():
        return kv0.clone(), l0.clone(), w0.clone()

    kv, lens, w = fresh()
    want_kept = F.evict_kv(kv, lens, w, cfg, 256, first=4, last=16)
    want = kv, lens, w
    state = fresh()
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        kept = F.evict_kv(*state, cfg, 256, first=4, last=16)
    for _ in range(3):
        for x, y in zip(state, (kv0, l0, w0)):
            x.copy_(y)
        graph.replay()
        side = fresh()
        F.evict_kv(*side, cfg, 300)
        torch.cuda.synchronize()
        assert torch.equal(kept, want_kept) and all(torch.equal(x, y) for x, y in zip(state, want))
    graph.replay()  # nothing is longer than it may be now
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(state, want))
    assert kept[0].tolist() == list(range(256)) and (kept[1] == -1).all()


def test_kept_is_optional_and_the_workspace_the_callers(cuda):
    lib = capi.load()
    g = torch.Generator().manual_seed(2)
    kv0, w0 = torch.randn(3, 300, 576, generator=g).bfloat16().to(cuda), torch.rand(3, 300, generator=g).to(cuda)
    l0 = torch.tensor([300, 20, 150], dtype=torch.int32, device=cuda)
    cfg = MLAConfig.deepseek_v2()
    kv, w, lens = kv0.clone(), w0.clone(), l0.clone()
    F.evict_kv(kv, lens, w, cfg, 100, first=2, last=3)
    for own in (True, False):
        x, y, z = kv0.clone(), w0.clone(), l0.clone()
        a = capi.EvictArgs(kv_cache=x.data_ptr(), kv_dtype=capi.LA_DTYPE_BF16, total_rows=900, num_seqs=3, seq_capacity=300,
                           seq_lens=z.data_ptr(), weights=y.data_ptr(), keep=100, first=2, last=3, cfg=capi.config(cfg))
        need = lib.la_evict_kv_workspace_size(ctypes.byref(a))
        assert need > 3 * 100 * 4
        ws = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device=cuda)
        if own:
            a.workspace, a.workspace_bytes = ws.data_ptr() + 8, need
        assert lib.la_evict_kv(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == capi.LA_SUCCESS
        torch.cuda.synchronize()
        assert torch.equal(x, kv) and torch.equal(y, w) and torch.equal(z, lens)
        assert (ws[need + 8:] == 0xFF).all() and (ws[:8] == 0xFF).all()


@pytest.mark.parametrize("keep", [300, 1 << 30])
def test_more_than_a_region_holds(cuda, keep):
    """Nothing can move: no workspace for it, whatever the number asked for."""
    lib = capi.load()
    g = torch.Generator().manual_seed(4)
    kv, w = torch.randn(3, 300, 576, generator=g).bfloat16().to(cuda), torch.rand(3, 300, generator=g).to(cuda)
    lens = torch.tensor([300, 20, 900], dtype=torch.int32, device=cuda)
    old = kv.clone(), w.clone(), lens.clone()
    a = capi.EvictArgs(kv_cache=kv.data_ptr(), kv_dtype=capi.LA_DTYPE_BF16, total_rows=900, num_seqs=3, seq_capacity=300,
                       seq_lens=lens.data_ptr(), weights=w.data_ptr(), keep=keep, cfg=capi.config(MLAConfig.deepseek_v2()))
    assert lib.la_evict_kv_workspace_size(ctypes.byref(a)) <= 4096
    assert lib.la_evict_kv(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == capi.LA_SUCCESS
    if keep == 300:
        kept = F.evict_kv(kv, lens, w, MLAConfig.deepseek_v2(), keep).cpu()
        for s, n in enumerate((300, 20, 300)):
            assert kept[s].tolist() == list(range(n)) + [-1] * (keep - n)
    assert torch.equal(kv, old[0]) and torch.equal(w, old[1]) and torch.equal(lens, old[2])


def test_few_and_many_sequences_agree(cuda):
    """A few sequences' rows go through a copy, many are moved where they lie: the same rows either way."""
    g = torch.Generator().manual_seed(6)
    cfg = MLAConfig.deepseek_v2()
    kv, w = torch.randn(64, 500, 576, generator=g).bfloat16().to(cuda), torch.rand(64, 500, generator=g).to(cuda)
    lens = torch.randint(300, 501, (64,), generator=g, dtype=torch.int32).to(cuda)
    one = [x.clone() for x in (kv, w, lens)]
    kept = F.evict_kv(kv, lens, w, cfg, 250, first=4, last=16)
    for s in (0, 31, 63):
        a, b, n = (x[s:s + 1].clone() for x in one)
        k = F.evict_kv(a, n, b, cfg, 250, first=4, last=16)
        assert torch.equal(k[0], kept[s]) and torch.equal(n[0], lens[s]) and torch.equal(b[0], w[s])
        assert torch.equal(a[0, :250], kv[s, :250])
