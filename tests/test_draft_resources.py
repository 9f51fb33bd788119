"""CPU check of the draft-tree and cache-cutting kernels as compiled (hipcc, gfx950 assembly): none spills to scratch, and
no instruction of the 128-head kernel's form for trees touches a register that an inline-asm read has not yet written
(tests/lds_wait_check.py)."""

from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

from lds_wait_check import kernels, kernels_with_labels, pending_uses, pending_uses_cfg

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
TREE = "_ZN2la12_GLOBAL__N_123decode_mfma_tree_kernel"


def assembly(source, tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    src = os.path.join(ROOT, "latent-attn_amd", "csrc")
    out = tmp_path / "kernels.s"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "-I", os.path.join(ROOT, "include"), "-I", src, "--cuda-device-only", "-S",
                    os.path.join(src, source + ".hip"), "-o", str(out)], check=True, capture_output=True, timeout=600)
    return out.read_text()


def check_scratch(text, least, only=""):
    sizes = {}
    for line in text.splitlines():
        if m := re.match(r"\s*\.amdhsa_kernel (\S+)", line):
            name = m.group(1)
        elif m := re.match(r"\s*\.amdhsa_private_segment_fixed_size (\d+)", line):
            sizes[name] = int(m.group(1))
    sizes = {n: b for n, b in sizes.items() if only in n}
    assert len(sizes) >= least
    assert {n: b for n, b in sizes.items() if b} == {}
    assert not re.search(r"v_pk_(add|mul|fma)_f32", text)


@pytest.mark.parametrize("source,least", [("la_tree", 4), ("la_weigh", 13), ("la_evict", 17)])
def test_no_scratch(source, least, tmp_path):
    check_scratch(assembly(source, tmp_path), least)


def test_attention_over_trees(tmp_path):
    text = assembly("la_mfma", tmp_path)
    check_scratch(text, 6, TREE)  # {bf16, f16, fp8} x {contiguous, paged}
    for parse, uses in ((kernels, pending_uses), (kernels_with_labels, pending_uses_cfg)):
        found = parse(text, TREE)
        assert len(found) == 6
        for name, instructions in found.items():
            assert uses(instructions) == [], name
