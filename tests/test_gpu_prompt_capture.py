"""The C entries of prompts, prefixes and shared steps under stream capture: with the caller's workspace they are recorded,
without one refused, and the graph gives the eager calls' bits on every replay."""

from __future__ import annotations

import ctypes

import pytest
import torch

from prompt_cases import tables, weights

from latent_attn import MLAConfig, capi

pytestmark = pytest.mark.gpu

HEADS, ROWS, TOKENS = 16, 130, 3


class Calls:
    """One sequence's prompt, an expansion of its rows and a step of two sequences behind them."""

    def __init__(self, cuda):
        g = torch.Generator().manual_seed(1)
        cfg = MLAConfig(5120, 512, 128, 64, HEADS, 128)
        self.lib, c = capi.load(), capi.config(cfg)
        self.kv = torch.randn(ROWS, 576, generator=g).bfloat16().to(cuda)
        self.own = torch.randn(2, 20, 576, generator=g).bfloat16().to(cuda)
        self.W = [w.to(cuda) for w in weights(HEADS, torch.bfloat16, 2)]
        self.tables = [t.to(cuda) for t in tables(ROWS + 20)]
        self.q = [torch.randn(TOKENS, HEADS, d, generator=g).to(cuda) for d in (128, 64)]
        self.out = [torch.empty(TOKENS, HEADS, 128, device=cuda),
                    torch.empty(self.lib.la_expanded_size(ROWS, ctypes.byref(c)), dtype=torch.uint8, device=cuda),
                    torch.empty(2, HEADS, 128, device=cuda)]
        bf16, f32 = capi.LA_DTYPE_BF16, capi.LA_DTYPE_F32
        same = dict(W_UK=self.W[0].data_ptr(), w_uk_dtype=bf16, W_UV=self.W[1].data_ptr(), w_uv_dtype=bf16,
                    rope_cos=self.tables[0].data_ptr(), rope_sin=self.tables[1].data_ptr(), rope_rows=ROWS + 20, cfg=c)
        q = dict(q_nope=self.q[0].data_ptr(), q_rope=self.q[1].data_ptr())
        self.args = [
            ("la_mla_prefill", capi.PrefillArgs(kv_cache=self.kv.data_ptr(), kv_dtype=bf16, total_rows=ROWS, num_seqs=1,
                                                seq_len=ROWS, tokens=TOKENS, q_dtype=f32, rotate_q=1,
                                                output=self.out[0].data_ptr(), out_dtype=f32, **q, **same)),
            ("la_expand_prefix", capi.ExpandArgs(kv_cache=self.kv.data_ptr(), kv_dtype=bf16, rows=ROWS,
                                                 expanded=self.out[1].data_ptr(), expanded_bytes=self.out[1].numel(), **same)),
            ("la_mla_decode_shared", capi.SharedArgs(
                own=capi.DecodeArgs(kv_cache=self.own.data_ptr(), kv_dtype=bf16, total_rows=40, num_seqs=2, seq_len=20,
                                    queries_per_seq=1, **q, **same),
                prefix=self.kv.data_ptr(), prefix_len=ROWS, expanded=self.out[1].data_ptr(),
                output=self.out[2].data_ptr(), out_dtype=f32, kernel_variant=2)),
        ]
        self.spaces = []
        for name, a in self.args:
            need = getattr(self.lib, name + "_workspace_size")(ctypes.byref(a))
            assert need > 0
            self.spaces.append(torch.empty(need, dtype=torch.uint8, device=cuda))

    def run(self, own_memory):
        status = []
        for (name, a), ws in zip(self.args, self.spaces):
            a.workspace, a.workspace_bytes = (None, 0) if own_memory else (ws.data_ptr(), ws.numel())
            status.append(getattr(self.lib, name)(ctypes.byref(a), torch.cuda.current_stream().cuda_stream))
        return status


def test_a_workspace_under_capture(cuda):
    c = Calls(cuda)
    assert c.run(own_memory=True) == c.run(own_memory=False) == [capi.LA_SUCCESS] * 3
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        refused = c.run(own_memory=True)
        status = c.run(own_memory=False)
    assert refused == [capi.LA_ERROR_WORKSPACE] * 3 and status == [capi.LA_SUCCESS] * 3
    for seed in (3, 4, 5):
        c.kv.copy_(torch.randn(c.kv.shape, generator=torch.Generator().manual_seed(seed)).bfloat16())
        for o in c.out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in c.out]
        assert c.run(own_memory=True) == [capi.LA_SUCCESS] * 3
        torch.cuda.synchronize()
        assert all(torch.equal(x, o) for x, o in zip(got, c.out))
        assert torch.isfinite(got[0]).all() and torch.isfinite(got[2]).all() and (got[0] != 0).any()
