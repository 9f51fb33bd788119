"""CPU checks of the draft-tree and eviction entry points: struct layouts, refusals (which come before any HIP call),
workspace sizes, and the references that the GPU tests use."""

from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from draft_cases import ancestors, evict_reference, tree

from latent_attn import MLAConfig, capi

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, UNSUPPORTED, OK = capi.LA_ERROR_INVALID_VALUE, capi.LA_ERROR_NOT_SUPPORTED, capi.LA_SUCCESS
FAKE = 0x1000


def test_ctypes_structs_match_the_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    structs = {"la_tree_args": capi.TreeArgs, "la_accept_args": capi.AcceptArgs, "la_weigh_args": capi.WeighArgs,
               "la_evict_args": capi.EvictArgs}
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


def args(cls, **kw):
    a = cls(kv_dtype=capi.LA_DTYPE_BF16, num_seqs=2, total_rows=128, cfg=capi.config(MLAConfig.deepseek_v2()))
    defaults = {"seq_len": 64, "seq_capacity": 64, "q_dtype": capi.LA_DTYPE_BF16, "w_uk_dtype": capi.LA_DTYPE_BF16,
                "w_uv_dtype": capi.LA_DTYPE_BF16, "out_dtype": capi.LA_DTYPE_BF16, "nodes": 4, "tokens_per_seq": 2, "keep": 16}
    pointers = ("kv_cache", "q_nope", "q_rope", "W_UK", "W_UV", "rope_cos", "rope_sin", "output", "parents", "path", "weights")
    fields = {f for f, _ in cls._fields_}
    for f, v in {**defaults, **dict.fromkeys(pointers, FAKE)}.items():
        if f in fields:
            setattr(a, f, v)
    if "seq_capacity" in fields:
        a.seq_lens = FAKE
    for k, v in kw.items():
        setattr(a, k, v)
    return a


CALLS = {"la_mla_decode_tree": capi.TreeArgs, "la_accept_kv": capi.AcceptArgs, "la_weigh_kv": capi.WeighArgs,
         "la_evict_kv": capi.EvictArgs}
EVERY = [{"num_seqs": -1}, {"total_rows": 127}, {"total_rows": -1}, {"kv_dtype": 9}, {"kv_dtype": -1}, {"kv_cache": 0},
         {"seq_offsets": FAKE, "total_rows": 1 << 31},
         {"block_table": FAKE, "seq_lens": FAKE, "block_size": 0, "blocks_per_seq": 2},
         {"block_table": FAKE, "seq_lens": FAKE, "block_size": 48, "blocks_per_seq": 2},
         {"block_table": FAKE, "seq_lens": FAKE, "block_size": 32, "blocks_per_seq": 0},
         {"block_table": FAKE, "seq_lens": FAKE, "block_size": 32, "blocks_per_seq": 1 << 27},
         {"block_table": FAKE, "seq_lens": FAKE, "block_size": 32, "blocks_per_seq": 2, "seq_offsets": FAKE},
         {"block_table": FAKE, "seq_lens": FAKE, "block_size": 32, "blocks_per_seq": 2, "total_rows": 0},
         {"block_table": FAKE, "seq_lens": 0, "block_size": 32, "blocks_per_seq": 2}]
QUERIES = [{"q_dtype": capi.LA_DTYPE_FP8_E4M3}, {"q_dtype": 5}, {"rotate_q": 2}, {"rotate_q": -1}, {"q_nope": 0}, {"q_rope": 0},
           {"W_UK": 0}, {"rope_cos": 0}, {"rope_sin": 0}, {"rope_rows": -1}, {"w_uk_dtype": capi.LA_DTYPE_FP8_E4M3},
           {"q_nope_token_stride": -8}, {"q_rope_head_stride": -8}, {"kernel_variant": 3}, {"kernel_variant": -1},
           {"num_seqs": 2 ** 31 - 1, "seq_len": 0}, {"num_seqs": 2 ** 28, "seq_len": 0}, {"seq_len": -1}]
BAD = ([(n, b) for n in CALLS for b in EVERY] + [(n, b) for n in ("la_mla_decode_tree", "la_weigh_kv") for b in QUERIES] +
       [("la_mla_decode_tree", b) for b in ({"nodes": 0}, {"nodes": 65}, {"nodes": -1}, {"parents": 0}, {"W_UV": 0}, {"output": 0},
                                            {"w_uv_dtype": 7}, {"out_dtype": capi.LA_DTYPE_FP8_E4M3}, {"out_dtype": -1})] +
       [("la_accept_kv", b) for b in ({"nodes": 0}, {"nodes": 65}, {"path": 0}, {"seq_lens": 0}, {"seq_capacity": -1})] +
       [("la_weigh_kv", b) for b in ({"tokens_per_seq": -1}, {"weights": 0})] +
       [("la_evict_kv", b) for b in ({"keep": -1}, {"first": -1}, {"last": -1}, {"first": 9, "last": 8}, {"weights": 0},
                                     {"seq_lens": 0}, {"seq_capacity": -1}, {"first": 2 ** 31 - 1, "last": 2 ** 31 - 1})])


@pytest.mark.parametrize("name,bad", BAD)
def test_refuses(name, bad):
    lib = capi.load()
    a = args(CALLS[name], **bad)
    assert getattr(lib, name)(ctypes.byref(a), None) == INVALID
    if name != "la_accept_kv":
        assert getattr(lib, name + "_workspace_size")(ctypes.byref(a)) == 0


@pytest.mark.parametrize("name", CALLS)
def test_refuses_bad_config_and_null(name):
    lib = capi.load()
    assert getattr(lib, name)(None, None) == INVALID
    for field, value in (("num_heads", 0), ("qk_rope_head_dim", 63), ("kv_lora_rank", -1)):
        a = args(CALLS[name])
        setattr(a.cfg, field, value)
        assert getattr(lib, name)(ctypes.byref(a), None) == INVALID


@pytest.mark.parametrize("name", CALLS)
def test_without_sequences_is_a_no_op(name):
    lib = capi.load()
    a = args(CALLS[name], num_seqs=0, kv_cache=0, total_rows=0)
    assert getattr(lib, name)(ctypes.byref(a), None) == OK


def test_weighing_without_tokens_is_a_no_op():
    lib = capi.load()
    a = args(capi.WeighArgs, tokens_per_seq=0, q_nope=0, weights=0)
    assert lib.la_weigh_kv(ctypes.byref(a), None) == OK and lib.la_weigh_kv_workspace_size(ctypes.byref(a)) == 0


@pytest.mark.parametrize("name", ["la_mla_decode_tree", "la_weigh_kv", "la_evict_kv"])
def test_refuses_a_small_workspace(name):
    lib = capi.load()
    a = args(CALLS[name])
    need = getattr(lib, name + "_workspace_size")(ctypes.byref(a))
    assert need > 0
    a.workspace, a.workspace_bytes = 1 << 20, need - 1
    assert getattr(lib, name)(ctypes.byref(a), None) == capi.LA_ERROR_WORKSPACE


@pytest.mark.parametrize("name", ["la_mla_decode_tree", "la_weigh_kv"])
def test_shapes_without_a_kernel(name):
    lib = capi.load()
    a = args(CALLS[name])
    a.cfg.kv_lora_rank = 2048
    assert getattr(lib, name)(ctypes.byref(a), None) == UNSUPPORTED
    a = args(CALLS[name], kernel_variant=2, kv_dtype=capi.LA_DTYPE_F32)
    assert getattr(lib, name)(ctypes.byref(a), None) == UNSUPPORTED


def test_references():
    assert ancestors([-1, 0, 0, 2, 9]) == [{0}, {0, 1}, {0, 2}, {0, 2, 3}, {4}]
    assert tree(4, 0, "chain") == [-1, 0, 1, 2] and all(-1 <= p < j for j, p in enumerate(tree(64, 1)))
    nan = float("nan")
    assert evict_reference([1, 5, 5, 2, 5, 0], 4, 1, 1) == [0, 1, 2, 5]
    assert evict_reference([nan, nan, 0, -1, nan], 3, 0, 0) == [0, 2, 3]
    assert evict_reference([-float("inf"), nan, 3], 2, 0, 0) == [0, 2]
    assert evict_reference([1, 2], 2, 0, 0) == [0, 1]
