"""evict_kv at the edges of its arguments' ranges."""

from __future__ import annotations

import pytest
import torch

from latent_attn import MLAConfig
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
