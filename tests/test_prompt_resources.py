"""CPU check of the prompt and shared-prefix kernels' registers: none spills to scratch, and two workgroups of the
prompt kernel fit a CU (hipcc, gfx950 assembly)."""

from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


@pytest.mark.parametrize("source,least", [("la_prompt", 6), ("la_expand", 17), ("la_join", 2)])
def test_no_scratch(source, least, tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    src = os.path.join(ROOT, "latent-attn_amd", "csrc")
    out = tmp_path / "kernels.s"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "-I", os.path.join(ROOT, "include"), "-I", src, "--cuda-device-only", "-S",
                    os.path.join(src, source + ".hip"), "-o", str(out)], check=True, capture_output=True, timeout=600)
    text = out.read_text()
    scratch, registers = {}, {}
    for line in text.splitlines():
        if m := re.match(r"\s*\.amdhsa_kernel (\S+)", line):
            name = m.group(1)
        elif m := re.match(r"\s*\.amdhsa_private_segment_fixed_size (\d+)", line):
            scratch[name] = int(m.group(1))
        elif m := re.match(r"\s*\.amdhsa_next_free_vgpr (\d+)", line):
            registers[name] = int(m.group(1))
    assert len(scratch) >= least
    assert {n: b for n, b in scratch.items() if b} == {}
    assert not re.search(r"v_pk_(add|mul|fma)_f32", text)
    for name, n in registers.items():
        # two waves per SIMD of 512 registers: two workgroups of 4 waves, or one of 8
        if "prompt_kernel" in name and "generic" not in name or "expand_kernel" in name:
            assert n <= 256, name
