"""evict_kv at the edges of its arguments' ranges."""

from __future__ import annotations

import ctypes

import pytest
import torch

from latent_attn import MLAConfig, capi
from latent_attn import functional as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("keep", [2 ** 31 - 1, 2 ** 31 - 700])
@pytest.mark.parametrize("region", [300, 5000])
def test_as_many_rows_as_a_number_holds(cuda, keep, region):
    """keep near 2^31: nothing can be cut; the list holds every row's position and -1 behind them, to its end (its counter
    passes 2^31 in the last step of 256 or 1024)."""
    g = torch.Generator().manual_seed(1)
    kv, w = torch.randn(1, region, 576, generator=g).bfloat16().to(cuda), torch.rand(1, region, generator=g).to(cuda)
    lens = torch.tensor([region - 7], dtype=torch.int32, device=cuda)
    old = kv.clone(), w.clone(), lens.clone()
    kept = F.evict_kv(kv, lens, w, MLAConfig.deepseek_v2(), keep, first=4, last=16)
    assert kept.shape == (1, keep)
    n = region - 7
    assert kept[0, :n].tolist() == list(range(n))
    for part in kept[0, n:].split(1 << 28):
        assert (part == -1).all()
    assert torch.equal(kv, old[0]) and torch.equal(w, old[1]) and torch.equal(lens, old[2])


@pytest.mark.parametrize("rows,keep", [(40000, 30000), (40000, 100), (20000, 19999), (5000, 2000)])
@pytest.mark.parametrize("seqs", [2, 15])
def test_packed_offsets_that_are_not_in_order(cuda, rows, keep, seqs):
    """Sequences that overlap move one another's rows and weights, so that a weight may be another one whenever it is read: what
    stays is anybody's guess, but every entry names a row of the cache and nothing is written beside the lists."""
    lib = capi.load()
    g = torch.Generator().manual_seed(1)
    kv, w = torch.randn(rows, 16, generator=g).bfloat16().to(cuda), torch.rand(rows + 64, generator=g).to(cuda)
    behind = w[rows:].clone()
    offsets = torch.tensor(([0, rows] * 8)[:seqs + 1], dtype=torch.int32, device=cuda)
    lens = torch.full((seqs,), rows, dtype=torch.int32, device=cuda)
    guard = seqs * rows  # more than all that could be listed
    kept = torch.full((seqs * keep + guard,), -7, dtype=torch.int32, device=cuda)
    a = capi.EvictArgs(kv_cache=kv.data_ptr(), kv_dtype=capi.LA_DTYPE_BF16, total_rows=rows, num_seqs=seqs,
                       seq_offsets=offsets.data_ptr(), seq_lens=lens.data_ptr(), weights=w.data_ptr(), keep=keep, first=4, last=16,
                       kept=kept.data_ptr(), cfg=capi.config(MLAConfig(5120, 12, 128, 4, 16, 128)))
    need = lib.la_evict_kv_workspace_size(ctypes.byref(a))
    ws = torch.full((need + 4 * guard,), 0xFF, dtype=torch.uint8, device=cuda)
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    assert lib.la_evict_kv(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == capi.LA_SUCCESS
    torch.cuda.synchronize()
    assert (kept[seqs * keep:] == -7).all() and (ws[need:] == 0xFF).all() and torch.equal(w[rows:], behind)
    listed = kept[:seqs * keep]
    assert ((listed >= -1) & (listed < rows)).all()
    assert kv.isfinite().all()
