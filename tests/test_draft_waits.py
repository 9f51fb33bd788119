"""CPU check of the compiled 128-head kernels for trees of drafted tokens: no instruction touches a register that an
inline-asm LDS read or vector-memory load has not yet written (tests/lds_wait_check.py), over both counters; and of what that
check takes for an unused high half."""

from __future__ import annotations

import pytest

from lds_wait_check import kernels, kernels_with_labels, pending_uses, pending_uses_cfg
from test_draft_resources import TREE, assembly

LOAD = "global_load_dword v205, v[0:1], off"
MAD = "v_mad_u64_u32 v[192:193], s[68:69], v192, s78, v[204:205]"


@pytest.mark.parametrize("uses", [pending_uses, pending_uses_cfg])
def test_a_high_half_that_an_lds_read_overwrites(uses):
    dead = [LOAD, MAD, "ds_read_b128 v[192:195], v216", "s_waitcnt vmcnt(0) lgkmcnt(0)", "v_mov_b32_e32 v7, v193"]
    assert uses(dead, counters=("lgkm", "vm")) == []
    # read, or stored, or an address, before it is overwritten
    for use in ("v_mov_b32_e32 v7, v193", "ds_write_b32 v5, v193", "ds_write_b32 v193, v5", "global_store_dword v193, v5, s[0:1]",
                "ds_read_b32 v7, v193"):
        assert [b[0] for b in uses(dead[:2] + [use] + dead[2:], counters=("lgkm", "vm"))] == [1], use
    # what overwrites it is another part of the register file, or a load that is itself pending
    assert [b[0] for b in uses([LOAD, MAD, "ds_read_b64 v[194:195], v216", "v_mov_b32_e32 v7, v193"], counters=("vm",))] == [1]
    early = dead[:3] + ["v_mov_b32_e32 v7, v193"]
    assert [b[0] for b in uses(early, counters=("lgkm", "vm"))] == [3]


def test_no_register_touched_before_its_wait(tmp_path):
    text = assembly("la_mfma", tmp_path)
    for parse, uses in ((kernels, pending_uses), (kernels_with_labels, pending_uses_cfg)):
        found = parse(text, TREE)
        assert len(found) == 6  # {bf16, f16, fp8} x {contiguous, paged}
        for name, instructions in found.items():
            assert uses(instructions, counters=("lgkm", "vm")) == [], name
