"""weigh_kv at the edges of its arguments' ranges: offsets that are not in order, rooms far wider than their rows,
queries outside fp16's range over an fp16 cache, queries that are not finite;
and what two fp16 parts keep."""

from __future__ import annotations

import ctypes

import pytest
import torch

from draft_cases import places, weight_places
from prompt_cases import tables, weights
from test_gpu_weigh import Case

from latent_attn import MLAConfig, capi

pytestmark = pytest.mark.gpu

MiB = 1 << 20


@pytest.mark.parametrize("tokens,heads", [(1, 16), (4, 128)])
@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("order", ["0n", "n0", "late"])
def test_packed_offsets_that_are_not_in_order(cuda, tokens, heads, variant, order):
    """Sequences that overlap have more tiles together than the cache has rows for: what they get is anybody's guess,
    but nothing is written beside the workspace. (Its guard is as large as all their scores.)"""
    lib, rows, seqs = capi.load(), 1024, 15
    at = {"0n": [0, rows] * 8, "n0": [rows, 0] * 8, "late": [0, 5, 40, rows, -7, rows, 3, 1 << 30, 0, 900, 0, rows, 1, rows, 0, rows]}[order]
    g = torch.Generator().manual_seed(1)
    kv = torch.randn(rows, 576, generator=g).bfloat16().to(cuda)
    q = torch.randn(seqs * tokens, heads, 192, generator=g).bfloat16().to(cuda)
    W_UK = weights(heads, torch.bfloat16, 2)[0].to(cuda)
    cos, sin = (x.to(cuda) for x in tables(rows))
    offsets = torch.tensor(at, dtype=torch.int32, device=cuda)
    w = torch.zeros(rows + 64, device=cuda)
    a = capi.WeighArgs(kv_cache=kv.data_ptr(), kv_dtype=capi.LA_DTYPE_BF16, total_rows=rows, num_seqs=seqs,
                       seq_offsets=offsets.data_ptr(), tokens_per_seq=tokens, q_nope=q.data_ptr(), q_rope=q.data_ptr() + 256,
                       q_dtype=capi.LA_DTYPE_BF16, q_nope_token_stride=heads * 192, q_nope_head_stride=192,
                       q_rope_token_stride=heads * 192, q_rope_head_stride=192, rotate_q=1, W_UK=W_UK.data_ptr(),
                       w_uk_dtype=capi.LA_DTYPE_BF16, rope_cos=cos.data_ptr(), rope_sin=sin.data_ptr(), rope_rows=rows,
                       weights=w.data_ptr(), cfg=capi.config(MLAConfig(5120, 512, 128, 64, heads, 128)), kernel_variant=variant)
    need = lib.la_weigh_kv_workspace_size(ctypes.byref(a))
    guard = seqs * (rows // 32 + 1) * (-(-tokens * heads // 32)) * 4096
    ws = torch.full((need + guard,), 0xFF, dtype=torch.uint8, device=cuda)
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    for _ in range(2):
        assert lib.la_weigh_kv(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == capi.LA_SUCCESS
    torch.cuda.synchronize()
    assert (ws[need:] == 0xFF).all() and (w[rows:] == 0).all()


def in_room(c, room, packed):
    """The case's sequences at the front of regions of `room` rows (packed: of one cache with offsets that far apart)."""
    count, device = len(c.rows), c.q.device
    kv = torch.zeros(count, room, 576, dtype=c.layout.kv.dtype, device=device)
    kv[:, :c.layout.kv.shape[1]] = c.layout.kv
    c.layout.kv = kv
    if packed:
        c.layout.kv = kv.view(-1, 576)
        c.layout.kw["seq_offsets"] = torch.arange(count + 1, dtype=torch.int32, device=device) * room
    c.weights = torch.rand(*(c.layout.kv.shape[:1] if packed else (count, room)), device=device)
    c.cos, c.sin = (x.to(device) for x in tables(room))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("tokens,heads,room,pieces", [(31, 128, 131072, 8), (5, 128, 1 << 20, 10), (7, 127, 400000, 7), (3, 129, 131072, 1)])
def test_windows_in_wide_rooms(cuda, packed, tokens, heads, room, pieces):
    """Windows of any number of tokens in several pieces, which may end between a token's heads."""
    c = Case(cuda, "capacity", [tokens + 90, 200], tokens, heads=heads, kv=torch.float8_e4m3fn, seed=tokens)
    in_room(c, room, packed)
    c.check(2, (tokens, heads, room, packed), pieces)


@pytest.mark.parametrize("tokens", [1, 5, 7, 8, 31, 32, 33, 100])
@pytest.mark.parametrize("heads", [1, 16, 65, 127, 128, 129, 5000])
@pytest.mark.parametrize("room", [131072, 1 << 20, 40 << 20])
@pytest.mark.parametrize("packed", [False, True])
def test_scores_take_no_more_than_they_may(cuda, tokens, heads, room, packed):
    """512 MiB of scores at a time, or those of 32 (token, head) rows: 128 B per row of room (packed: and 4 KiB per
    sequence). The rest: two 16-bit parts of 576 elements per query row, their rows in whole 32 per sequence, and for up to
    512 workgroups and 4 sequences partial sums of 8 B for 4096 rows at most."""
    lib, seqs, fake = capi.load(), 4, 1 << 12
    a = capi.WeighArgs(kv_cache=fake, kv_dtype=capi.LA_DTYPE_BF16, total_rows=seqs * room, num_seqs=seqs, seq_len=room, seq_lens=fake,
                       tokens_per_seq=tokens, q_nope=fake, q_rope=fake, q_dtype=capi.LA_DTYPE_BF16, rotate_q=1, W_UK=fake,
                       w_uk_dtype=capi.LA_DTYPE_BF16, rope_cos=fake, rope_sin=fake, rope_rows=room, weights=fake,
                       cfg=capi.config(MLAConfig(5120, 512, 128, 64, heads, 128)), kernel_variant=2)
    if packed:
        a.seq_len, a.seq_offsets = 0, fake
    need = lib.la_weigh_kv_workspace_size(ctypes.byref(a))
    queries = seqs * -(-tokens * heads // 32) * 32 * 2 * 576 * 2
    least = 128 * seqs * room + 4096 * seqs if packed else 128 * room
    assert 0 < need <= max(512 * MiB, least) + queries + 516 * 4096 * 8 + 4096


def large(c, what, up):
    """Queries far past fp16's range (or far below one) over rows that are as much smaller (larger), so that scores stay where
    they were: all of them, one latent column in every head, the rope part, or a few heads' (whose scores move then)."""
    q, kv = c.q.clone(), c.layout.kv.float()
    if what == "all":
        q, kv = q * up, kv / up
    elif what == "column":
        c.W_UK[:, 100] *= up
        kv[..., 100] /= up
    elif what == "rope":
        q[..., 128:] *= up
        kv[..., 512:] /= up
    elif what == "edge":  # keys that pass fp16's range when they are rotated
        q[..., 128:] /= up
        kv[..., 512:] = (kv[..., 512:] * 2 * up).clamp(-65504, 65504)
    else:
        q[::2, ::5] *= up
    c.q, c.layout.kv = q, kv.to(c.layout.kv.dtype)
    flat = c.layout.kv.view(-1, 576).cpu().double()
    c.rows = [flat[places(c.layout, s, len(r))] for s, r in enumerate(c.rows)]


@pytest.mark.parametrize("what,up", [(x, y) for x in ("all", "column", "rope", "some") for y in (2.0 ** 10, 2.0 ** 14, 2.0 ** -12)] +
                         [("edge", 2.0 ** 15)])
@pytest.mark.parametrize("tokens,heads", [(1, 16), (3, 16), (3, 128), (2, 3)])
@pytest.mark.parametrize("w", [torch.bfloat16, torch.float32])
def test_large_queries_over_an_fp16_cache(cuda, what, up, tokens, heads, w):
    """Absorbed and scaled, elements of up to some 10^4 (q 2^14, scale log2(e) 0.1): fp16 holds 64 times them up to 1023. With
    float32 weights the operands come from another kernel."""
    c = Case(cuda, "paged", [70, 9, 300], tokens, heads=heads, kv=torch.float16, q=torch.float32, w=w, seed=5)
    large(c, what, up)
    for variant in (2, 1):
        c.check(variant, (what, up, variant))


@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("part", [slice(5, 6), slice(150, 151), slice(0, 192)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("tokens,heads", [(3, 16), (40, 16), (5, 128)])
def test_a_query_that_is_not_finite_stays_with_the_rows_it_sees(cuda, variant, kv, part, bad, tokens, heads):
    """One head of one token, in a sequence between two others: the rows behind the token get what the others give them."""
    c = Case(cuda, "paged", [50, 130, 70], tokens, heads=heads, kv=kv, seed=7)
    c.q[tokens + 1, heads // 2, part] = bad  # the second token of the second sequence: it sees rows 0 to 130 - tokens + 1
    w = torch.zeros_like(c.weights)
    c.run(w, kernel_variant=variant)
    got = w.cpu().double().view(-1)
    ref, bounds, _ = c.reference()
    for s, (r, b) in enumerate(zip(ref, bounds)):
        at = weight_places(c.layout, s, len(r))
        seen = torch.arange(len(r)) < (130 - tokens + 2 if s == 1 else 0)
        assert got[at][seen].isnan().all() and r[~seen].isfinite().all()
        assert ((got[at] - r).abs()[~seen] <= b[~seen]).all()


@pytest.mark.parametrize("kv", [torch.float8_e4m3fn, torch.float16])
@pytest.mark.parametrize("tokens,heads", [(1, 16), (1, 64), (1, 128), (16, 16)])
@pytest.mark.parametrize("w", [torch.bfloat16, torch.float32])
def test_fp16_parts_keep_as_much_as_fp32(cuda, kv, tokens, heads, w):
    """Over fp16 and 8-bit rows, which fp16 holds exactly, two fp16 parts of a query are off by 2^-23 of it (11 bits each), a
    score of about B = 1 (the root of its terms' squares) by no more; its fp32 sum of some 80 steps by 9 half steps of 2^-24
    (roundings are independent), 2^-22 together with the exponential's. A weight moves by twice that, its exponent's and its
    sum's: 2 (2^-23 + 2^-22) < 2^-20. Two bf16 parts left 2^-18 of a query."""
    c = Case(cuda, "paged", [300, 1500], tokens, heads=heads, kv=kv, q=torch.float32, w=w, seed=9)
    weight = torch.zeros_like(c.weights)
    c.run(weight, kernel_variant=2)
    got = weight.cpu().double().view(-1)
    for s, r in enumerate(c.reference()[0]):
        at = weight_places(c.layout, s, len(r))
        assert (got[at] - r).norm() <= 2.0 ** -20 * r.norm()


@pytest.mark.parametrize("q", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("up", [1.0, 2.0 ** 14, 2.0 ** 20, 2.0 ** -14])
@pytest.mark.parametrize("kv", [torch.float16, torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("tokens,heads,some", [(1, 16, False), (3, 128, False), (70, 16, True)])
def test_large_queries_with_fp16_weights(cuda, q, up, kv, tokens, heads, some):
    """Queries that fp16 does not hold against an fp16 W_UK whose columns are as much smaller (2^-14 at least: fp16's own
    range; the rope part is as it was). some: of every other token alone, whose scores grow."""
    c = Case(cuda, "capacity", [70 + tokens, 9, 200], tokens, heads=heads, kv=kv, q=q, w=torch.float16, seed=5)
    c.q[:: 2 if some else 1, :, :128] *= up
    if not some:
        c.W_UK = (c.W_UK.float() / min(max(up, 2.0 ** -10), 2.0 ** 10)).half()
        if up > 2.0 ** 10:
            c.q[..., :128:2] = 0  # (the scores grow by what the weights cannot take back)
    for variant in (2, 1):
        if some and up > 2.0 ** 14:
            # scores of 10^6, whose error leaves open which of two close ones is the larger (the bound of a weight is without
            # limit, and not a number where the weight is 0): each token's and head's weights still add up to 1, in sums of as
            # many terms as there are tokens, heads and rows, and each is 0 or more
            w = torch.zeros_like(c.weights)
            c.run(w, kernel_variant=variant)
            for s, r in enumerate(c.rows):
                got = w[s, :len(r)].double()
                ones = heads * min(tokens, len(r))
                assert (got >= 0).all() and abs(float(got.sum()) - ones) <= (ones + len(r) + 16) * 2.0 ** -24 * ones
        else:
            c.check(variant, (up, variant))
    if not some:  # queries out of line: absorbed apart
        pad = torch.zeros(*c.q.shape[:2], c.q.shape[2] + 1, dtype=q, device=cuda)
        pad[..., 1:] = c.q
        c.q = pad[..., 1:]
        c.check(2, (up, "out of line"))


@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("part", [slice(300, 301), slice(540, 541), slice(575, 576)])
def test_one_element_of_a_row_that_is_not_a_number(cuda, variant, kv, part):
    """Of every type, in the latent or the rope part: its own sequence's weights, and no other's."""
    c = Case(cuda, "paged", [50, 60, 70], 3, kv=kv, seed=3)
    ref, bounds, _ = c.reference()
    flat = c.layout.kv.view(-1, 576)
    where = places(c.layout, 1, 60)[20]
    row = flat[where].float()
    row[part] = float("nan")
    flat[where] = row.to(kv)
    w = torch.zeros_like(c.weights)
    c.run(w, kernel_variant=variant)
    got = w.cpu().double().view(-1)
    assert got[weight_places(c.layout, 1, 60)].isnan().all()
    for s in (0, 2):
        assert ((got[weight_places(c.layout, s, len(ref[s]))] - ref[s]).abs() <= bounds[s]).all()
