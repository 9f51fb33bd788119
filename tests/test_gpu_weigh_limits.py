"""weigh_kv at the edges of its arguments' ranges: offsets that are not in order."""

from __future__ import annotations

import ctypes

import pytest
import torch

from prompt_cases import tables, weights

from latent_attn import MLAConfig, capi

pytestmark = pytest.mark.gpu


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
