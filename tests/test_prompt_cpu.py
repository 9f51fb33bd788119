"""CPU checks of the prompt and shared-prefix entry points: struct layouts,
refusals (which come before any HIP call) and workspace sizes."""

from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from latent_attn import MLAConfig, capi
from latent_attn import functional as F

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, UNSUPPORTED, OK = capi.LA_ERROR_INVALID_VALUE, capi.LA_ERROR_NOT_SUPPORTED, capi.LA_SUCCESS
FAKE = 0x1000


def test_ctypes_structs_match_the_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    structs = {"la_prefill_args": capi.PrefillArgs, "la_expand_args": capi.ExpandArgs, "la_shared_args": capi.SharedArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "latent_attn.h"', "int main(void) {"]
    want = []
    for c, py in structs.items():
        lines.append(f'  printf("{c} size %zu\\n", sizeof({c}));')
        want.append(f"{c} size {ctypes.sizeof(py)}")
        for f, _ in py._fields_:
            lines.append(f'  printf("{c} {f} %zu\\n", offsetof({c}, {f}));')
            want.append(f"{c} {f} {getattr(py, f).offset}")
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run([gcc, "-I" + os.path.join(REPO, "include"), str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines() == want


def prefill_args(**kw):
    a = capi.PrefillArgs(kv_dtype=capi.LA_DTYPE_BF16, num_seqs=2, seq_len=64, total_rows=128, tokens=8,
                         q_dtype=capi.LA_DTYPE_BF16, w_uk_dtype=capi.LA_DTYPE_BF16, w_uv_dtype=capi.LA_DTYPE_BF16,
                         out_dtype=capi.LA_DTYPE_BF16, cfg=capi.config(MLAConfig.deepseek_v2()))
    for f in ("kv_cache", "q_nope", "q_rope", "W_UK", "W_UV", "rope_cos", "rope_sin", "output"):
        setattr(a, f, FAKE)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [
    {"num_seqs": -1}, {"tokens": -1}, {"tokens": 7}, {"total_rows": 127}, {"total_rows": -1}, {"seq_len": -1},
    {"rope_rows": -1}, {"max_seq_rows": -1}, {"kernel_variant": 4}, {"kernel_variant": -1}, {"rotate_q": 2},
    {"kv_dtype": 9}, {"q_dtype": capi.LA_DTYPE_FP8_E4M3}, {"q_dtype": 5}, {"out_dtype": capi.LA_DTYPE_FP8_E4M3},
    {"out_dtype": -1}, {"w_uk_dtype": capi.LA_DTYPE_FP8_E4M3}, {"w_uv_dtype": 7}, {"num_seqs": 0},
    {"kv_cache": 0}, {"q_nope": 0}, {"q_rope": 0}, {"W_UK": 0}, {"W_UV": 0}, {"rope_cos": 0}, {"rope_sin": 0},
    {"output": 0}, {"q_nope_token_stride": -8}, {"q_rope_head_stride": -8}, {"tokens": 1 << 40},
    {"num_seqs": 2 ** 31 - 1, "seq_len": 0},
    {"seq_offsets": FAKE, "max_seq_rows": 8}, {"seq_offsets": FAKE, "total_rows": 1 << 31},
    {"block_table": FAKE, "block_size": 32, "blocks_per_seq": 2},                       # no seq_lens
    {"block_table": FAKE, "seq_lens": FAKE, "block_size": 0, "blocks_per_seq": 2},
    {"block_table": FAKE, "seq_lens": FAKE, "block_size": 48, "blocks_per_seq": 2},     # pool of 128 rows
    {"block_table": FAKE, "seq_lens": FAKE, "block_size": 32, "blocks_per_seq": 0},
    {"block_table": FAKE, "seq_lens": FAKE, "block_size": 32, "blocks_per_seq": 1 << 27},
    {"block_table": FAKE, "seq_lens": FAKE, "block_size": 32, "blocks_per_seq": 2, "seq_offsets": FAKE},
    {"block_table": FAKE, "seq_lens": FAKE, "block_size": 32, "blocks_per_seq": 2, "total_rows": 0},
])
def test_prefill_refuses(bad):
    lib = capi.load()
    a = prefill_args(**bad)
    assert lib.la_mla_prefill(ctypes.byref(a), None) == INVALID
    assert lib.la_mla_prefill_workspace_size(ctypes.byref(a)) == 0


def test_prefill_refuses_bad_config_and_null():
    lib = capi.load()
    assert lib.la_mla_prefill(None, None) == INVALID and lib.la_mla_prefill_workspace_size(None) == 0
    for field, value in (("num_heads", 0), ("qk_rope_head_dim", 63), ("kv_lora_rank", -1)):
        a = prefill_args()
        setattr(a.cfg, field, value)
        assert lib.la_mla_prefill(ctypes.byref(a), None) == INVALID


@pytest.mark.parametrize("why", [
    {"kernel_variant": 3, "seq_offsets": FAKE},                        # packed sequences have no block table
    {"kernel_variant": 2, "kv_dtype": capi.LA_DTYPE_F32},              # 16-bit operands only
    {"kernel_variant": 2, "output": FAKE + 2},                         # stores of 8 bytes
])
def test_prefill_forms_without_a_kernel(why):
    lib = capi.load()
    a = prefill_args(**why)
    assert lib.la_mla_prefill(ctypes.byref(a), None) == UNSUPPORTED
    a = prefill_args(kernel_variant=1)
    a.cfg.kv_lora_rank = 2048
    assert lib.la_mla_prefill(ctypes.byref(a), None) == UNSUPPORTED


def test_prefill_without_tokens_is_a_no_op():
    lib = capi.load()
    a = prefill_args(tokens=0, q_nope=0, output=0, kv_cache=0)
    assert lib.la_mla_prefill(ctypes.byref(a), None) == OK
    assert lib.la_mla_prefill_workspace_size(ctypes.byref(a)) == 0


def test_prefill_refuses_a_small_workspace():
    lib = capi.load()
    for variant in (1, 3):
        a = prefill_args(kernel_variant=variant)
        need = lib.la_mla_prefill_workspace_size(ctypes.byref(a))
        assert need > 0
        a.workspace, a.workspace_bytes = 1 << 20, need - 1
        assert lib.la_mla_prefill(ctypes.byref(a), None) == capi.LA_ERROR_WORKSPACE


def expand_args(**kw):
    a = capi.ExpandArgs(kv_dtype=capi.LA_DTYPE_BF16, rows=100, w_uk_dtype=capi.LA_DTYPE_BF16,
                        w_uv_dtype=capi.LA_DTYPE_BF16, cfg=capi.config(MLAConfig.deepseek_v2()), expanded=FAKE,
                        expanded_bytes=1 << 40)
    for f in ("kv_cache", "W_UK", "W_UV", "rope_cos", "rope_sin"):
        setattr(a, f, FAKE)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [
    {"rows": -1}, {"rope_rows": -1}, {"kv_dtype": 9}, {"w_uk_dtype": capi.LA_DTYPE_FP8_E4M3}, {"w_uv_dtype": 6},
    {"kv_cache": 0}, {"W_UK": 0}, {"W_UV": 0}, {"rope_cos": 0}, {"rope_sin": 0}, {"expanded": 0},
    {"expanded": FAKE + 16}, {"expanded_bytes": 1000},
])
def test_expand_refuses(bad):
    lib = capi.load()
    assert lib.la_expand_prefix(ctypes.byref(expand_args(**bad)), None) == INVALID


def test_expand_sizes_and_unsupported():
    lib = capi.load()
    cfg = capi.config(MLAConfig.deepseek_v2())
    assert lib.la_expanded_size(0, ctypes.byref(cfg)) == 0
    assert lib.la_expanded_size(1, ctypes.byref(cfg)) == lib.la_expanded_size(64, ctypes.byref(cfg)) == 64 * (128 * 512 + 128)
    assert lib.la_expanded_size(65, ctypes.byref(cfg)) == 128 * (128 * 512 + 128)
    assert lib.la_expanded_size(-1, ctypes.byref(cfg)) == 0 and lib.la_expanded_size(8, None) == 0
    other = capi.config(MLAConfig(5120, 256, 128, 64, 8, 128))
    assert lib.la_expanded_size(8, ctypes.byref(other)) == 0
    assert lib.la_expand_prefix(ctypes.byref(expand_args(cfg=other)), None) == UNSUPPORTED
    assert lib.la_expand_prefix(ctypes.byref(expand_args(kv_dtype=capi.LA_DTYPE_F32)), None) == UNSUPPORTED
    assert lib.la_expand_prefix(None, None) == INVALID
    assert lib.la_expand_prefix(ctypes.byref(expand_args(rows=0, expanded=0)), None) == OK


def shared_args(**kw):
    d = capi.DecodeArgs(kv_dtype=capi.LA_DTYPE_BF16, num_seqs=2, seq_len=16, total_rows=32, queries_per_seq=1,
                        w_uk_dtype=capi.LA_DTYPE_BF16, w_uv_dtype=capi.LA_DTYPE_BF16,
                        cfg=capi.config(MLAConfig.deepseek_v2()))
    for f in ("kv_cache", "q_nope", "q_rope", "W_UK", "W_UV", "rope_cos", "rope_sin"):
        setattr(d, f, FAKE)
    a = capi.SharedArgs(prefix=FAKE, prefix_len=100, output=FAKE, out_dtype=capi.LA_DTYPE_BF16)
    for k, v in kw.items():
        setattr(d if k.startswith("own_") else a, k.removeprefix("own_"), v)
    a.own = d
    return a


@pytest.mark.parametrize("bad", [
    {"prefix": 0}, {"prefix_len": -1}, {"output": 0}, {"out_dtype": capi.LA_DTYPE_FP8_E4M3}, {"kernel_variant": 3},
    {"own_num_seqs": -1}, {"own_queries_per_seq": 0}, {"own_q_nope": 0}, {"own_q_absorbed": FAKE}, {"own_q_rope": 0},
    {"own_W_UK": 0}, {"own_W_UV": 0}, {"own_rope_cos": 0}, {"own_rope_sin": 0}, {"own_rope_rows": -1},
    {"own_total_rows": 31}, {"own_kv_dtype": 9}, {"own_kv_cache": 0}, {"own_w_uv_dtype": 8},
    {"own_num_seqs": 2 ** 30, "own_seq_len": 0}, {"own_block_table": FAKE, "own_block_size": 16, "own_blocks_per_seq": 1},
])
def test_shared_refuses(bad):
    lib = capi.load()
    a = shared_args(**bad)
    assert lib.la_mla_decode_shared(ctypes.byref(a), None) == INVALID
    assert lib.la_mla_decode_shared_workspace_size(ctypes.byref(a)) == 0


def test_shared_unsupported_small_workspace_and_empty():
    lib = capi.load()
    assert lib.la_mla_decode_shared(None, None) == INVALID
    assert lib.la_mla_decode_shared(ctypes.byref(shared_args(kernel_variant=2)), None) == UNSUPPORTED  # not expanded
    a = shared_args()
    need = lib.la_mla_decode_shared_workspace_size(ctypes.byref(a))
    assert need > 0
    a.workspace, a.workspace_bytes = 1 << 20, need - 1
    assert lib.la_mla_decode_shared(ctypes.byref(a), None) == capi.LA_ERROR_WORKSPACE
    assert lib.la_mla_decode_shared(ctypes.byref(shared_args(own_num_seqs=0, output=0)), None) == OK


def test_extension_refuses_cpu_tensors_and_bad_shapes():
    cfg = MLAConfig(5120, 512, 128, 64, 4, 128)
    kv, q = torch.zeros(2, 8, 576, dtype=torch.bfloat16), torch.zeros(4, 4, 192, dtype=torch.bfloat16)
    W, t = torch.zeros(512, 512, dtype=torch.bfloat16), torch.zeros(8, 32)
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        F.mla_prefill(kv, q[..., :128], q[..., 128:], W, W, t, t, cfg)
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        F.expand_prefix(kv[0], W, W, t, t, cfg)
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        F.mla_decode_shared(kv[0], kv, q[:2, :, :128].float(), q[:2, :, 128:].float(), W, W, t, t, cfg)
    with pytest.raises(ValueError, match="expanded for 8 heads"):
        F.mla_decode_shared(F.SharedPrefix(kv[0], torch.zeros(0), 8), kv, q, q, W, W, t, t, cfg)


def test_shared_prefix_views():
    """The views put the library's order back into rows, heads and dims."""
    rows, heads = 70, 3
    tiles = 2
    flat = torch.arange(tiles * 64 * (2 * heads * 128 + 64))
    p = F.SharedPrefix(torch.zeros(rows, 576), flat, heads)
    k = p.k_nope.reshape(-1, heads, 128)
    v = p.v.reshape(-1, heads, 128)
    r = p.k_rope.reshape(-1, 64)
    assert k.shape == v.shape == (128, 3, 128) and r.shape == (128, 64)
    for row, h, d in ((0, 0, 0), (69, 2, 127), (33, 1, 77), (100, 0, 20)):
        t, i = divmod(row, 64)
        g, hi, lo = (d >> 2) & 1, (d >> 3) & 1, d & 3
        at = (((h * tiles + t) * 2 + i // 32) * 8 + d // 16) * 512 + 8 * (i % 32 + 32 * g) + 4 * hi + lo
        assert k[row, h, d] == at
        g, hi, lo = (i >> 2) & 1, (i >> 3) & 1, i & 3
        at = heads * tiles * 8192 + (((h * tiles + t) * 4 + d // 32) * 4 + i // 16) * 512 + 8 * (d % 32 + 32 * g) + 4 * hi + lo
        assert v[row, h, d] == at
        if d < 64:
            g, hi, lo = (d >> 2) & 1, (d >> 3) & 1, d & 3
            at = 2 * heads * tiles * 8192 + ((t * 2 + i // 32) * 4 + d // 16) * 512 + 8 * (i % 32 + 32 * g) + 4 * hi + lo
            assert r[row, d] == at
