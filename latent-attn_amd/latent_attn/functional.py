"""Stateless functional API for the MLA decode kernels.

Same entry points and argument order as the reference
(latent_attn/functional.py:24-116 in the reference repo): ``fused_mla``,
``naive_mla``, ``batched_fused_mla``; plus ``mla_decode`` (per-sequence and
ragged caches with query absorption, split-KV and the W_UV projection in one
call) and ``absorb_q``; ``append_kv``; ``mla_prefill`` (several new tokens per
sequence: prompts, chunks, drafted tokens), ``expand_prefix`` and
``mla_decode_shared`` (decode behind one prefix of the whole batch). All compute runs in the HIP library; nothing here
falls back to PyTorch math -- if the extension is missing, the call raises.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import TYPE_CHECKING, Optional, Union

import torch

if TYPE_CHECKING:
    from latent_attn import MLAConfig


def _load_ext():
    try:
        from latent_attn import _C

        return _C
    except ImportError as e:  # reference functional.py:13-21
        raise ImportError(
            "latent_attn C extension not found. "
            "Run `python latent-attn_amd/build.py` from the repo root to build it."
        ) from e


def _cfg_args(cfg: "MLAConfig"):
    return (cfg.d_model, cfg.kv_lora_rank, cfg.qk_nope_head_dim, cfg.qk_rope_head_dim, cfg.num_heads, cfg.v_head_dim)


def fused_mla(
    kv_cache: torch.Tensor,
    q_absorbed: torch.Tensor,
    q_rope: torch.Tensor,
    W_UV: torch.Tensor,
    rope_cos: torch.Tensor,
    rope_sin: torch.Tensor,
    cfg: "MLAConfig",
) -> torch.Tensor:
    """Single-token fused absorbed MLA forward.

    Args:
        kv_cache:   (seq_len, kv_lora_rank + qk_rope_head_dim) fp16 / bf16 / fp32
        q_absorbed: (num_heads, kv_lora_rank) fp32
        q_rope:     (num_heads, qk_rope_head_dim) fp32, already rotated
        W_UV:       (num_heads * v_head_dim, kv_lora_rank) fp16 / bf16 / fp32
        rope_cos:   (seq_len, qk_rope_head_dim // 2) fp32
        rope_sin:   (seq_len, qk_rope_head_dim // 2) fp32
        cfg:        MLAConfig

    Returns:
        (num_heads, v_head_dim) fp32
    """
    _C = _load_ext()
    return _C.fused_mla_forward(kv_cache, q_absorbed, q_rope, W_UV, rope_cos, rope_sin, *_cfg_args(cfg))


def naive_mla(
    kv_cache: torch.Tensor,
    W_UK: torch.Tensor,
    W_UV: torch.Tensor,
    q_nope: torch.Tensor,
    q_rope: torch.Tensor,
    rope_cos: torch.Tensor,
    rope_sin: torch.Tensor,
    cfg: "MLAConfig",
) -> torch.Tensor:
    """Single-token MLA forward from the un-absorbed query (q_nope, W_UK).

    Returns the decompress-then-attend result (num_heads, v_head_dim) fp32,
    computed on the GPU by la_naive_mla: K_nope = c_t W_UK^T and V = c_t
    W_UV^T in fp32, RoPE on k_rope, softmax, P V -- independent of the
    absorbed kernels (reference tests/test_python.py:26-63).
    """
    _C = _load_ext()
    return _C.naive_mla_forward(kv_cache, W_UK, W_UV, q_nope, q_rope, rope_cos, rope_sin, *_cfg_args(cfg))


def batched_fused_mla(
    kv_cache: torch.Tensor,
    q_absorbed: torch.Tensor,
    q_rope: torch.Tensor,
    W_UV: torch.Tensor,
    rope_cos: torch.Tensor,
    rope_sin: torch.Tensor,
    cfg: "MLAConfig",
) -> torch.Tensor:
    """Batched fused absorbed MLA forward over multiple tokens sharing one KV cache.

    Args:
        kv_cache:   (seq_len, kv_lora_rank + qk_rope_head_dim)
        q_absorbed: (batch, num_heads, kv_lora_rank) fp32
        q_rope:     (batch, num_heads, qk_rope_head_dim) fp32
        W_UV:       (num_heads * v_head_dim, kv_lora_rank)
        rope_cos / rope_sin: (seq_len, qk_rope_head_dim // 2) fp32

    Returns:
        (batch, num_heads, v_head_dim) fp32
    """
    _C = _load_ext()
    return _C.batched_fused_mla_forward(kv_cache, q_absorbed, q_rope, W_UV, rope_cos, rope_sin, *_cfg_args(cfg))


def mla_decode(
    kv_cache: torch.Tensor,
    q_nope: torch.Tensor,
    q_rope: torch.Tensor,
    W_UK: torch.Tensor,
    W_UV: torch.Tensor,
    rope_cos: torch.Tensor,
    rope_sin: torch.Tensor,
    cfg: "MLAConfig",
    seq_offsets: Optional[torch.Tensor] = None,
    chunk_rows: int = 0,
    kernel_variant: int = 0,
    seq_lens: Optional[torch.Tensor] = None,
    block_table: Optional[torch.Tensor] = None,
    block_size: int = 0,
) -> torch.Tensor:
    """One decode step for a batch of sequences, each with its own cache.

    Args:
        kv_cache:    (batch, seq_len, dc + dR) when ``seq_offsets`` is None, else
                     a packed (total_rows, dc + dR) cache
        q_nope:      (batch, num_heads, qk_nope_head_dim) fp32
        q_rope:      (batch, num_heads, qk_rope_head_dim) fp32, already rotated
        W_UK, W_UV:  (num_heads * {qk_nope,v}_head_dim, kv_lora_rank)
        rope_cos / rope_sin: (>= longest sequence, qk_rope_head_dim // 2) fp32,
                     indexed by the position inside each sequence
        seq_offsets: optional int32 (batch + 1,) device tensor; sequence b is
                     rows [seq_offsets[b], seq_offsets[b+1])
        chunk_rows, kernel_variant: tuning overrides (0 = automatic; variant
                     1 = VALU kernel, 2 = MFMA kernel)
        seq_lens:    optional int32 (batch,) device tensor; sequence b is the
                     first seq_lens[b] rows of its region (a capacity cache
                     filled by ``append_kv``)
        block_table, block_size: optional paged cache: kv_cache is a pool of
                     (num_blocks * block_size, dc + dR) rows and position p of
                     sequence b lives in row block_table[b, p // block_size] *
                     block_size + p % block_size (int32 (batch, blocks_per_seq)
                     device tensor; needs seq_lens)

    Returns:
        (batch, num_heads, v_head_dim) fp32
    """
    _C = _load_ext()
    return _C.mla_decode_forward(kv_cache, q_nope, q_rope, W_UK, W_UV, rope_cos, rope_sin, seq_offsets,
                                 *_cfg_args(cfg), chunk_rows, kernel_variant, seq_lens, block_table, block_size)


def mla_decode_absorbed(
    kv_cache: torch.Tensor,
    q_absorbed: torch.Tensor,
    q_rope: torch.Tensor,
    W_UV: torch.Tensor,
    rope_cos: torch.Tensor,
    rope_sin: torch.Tensor,
    cfg: "MLAConfig",
    seq_offsets: Optional[torch.Tensor] = None,
    seq_lens: Optional[torch.Tensor] = None,
    chunk_rows: int = 0,
    kernel_variant: int = 0,
    block_table: Optional[torch.Tensor] = None,
    block_size: int = 0,
) -> torch.Tensor:
    """``mla_decode`` for queries already in latent space: q_absorbed
    (batch, num_heads, kv_lora_rank) fp32 (e.g. x . W_Q_absorbed^T). Same
    cache / sequence arguments; returns (batch, num_heads, v_head_dim) fp32."""
    _C = _load_ext()
    return _C.mla_decode_absorbed_forward(kv_cache, q_absorbed, q_rope, W_UV, rope_cos, rope_sin, seq_offsets,
                                          *_cfg_args(cfg), chunk_rows, kernel_variant, seq_lens, block_table,
                                          block_size)


def append_kv(
    kv_cache: torch.Tensor,
    seq_lens: torch.Tensor,
    c_t: torch.Tensor,
    k_rope: torch.Tensor,
    cfg: "MLAConfig",
    q_rope: Optional[torch.Tensor] = None,
    rope_cos: Optional[torch.Tensor] = None,
    rope_sin: Optional[torch.Tensor] = None,
    seq_offsets: Optional[torch.Tensor] = None,
    status: Optional[torch.Tensor] = None,
    block_table: Optional[torch.Tensor] = None,
    block_size: int = 0,
) -> None:
    """Append new latent rows to every sequence's cache on the device.

    The device-side counterpart of the reference's
    ``LatentKVCache::append_host`` (src/mla_config.cuh:57-72) for a batch:
    no host copies and no synchronize; lengths are kept on the device.

    Args:
        kv_cache:    (batch, capacity, dc + dR) when ``seq_offsets`` is None,
                     else a packed (rows, dc + dR) cache whose sequence b owns
                     rows [seq_offsets[b], seq_offsets[b+1])
        seq_lens:    int32 (batch,) device tensor of filled rows, advanced in
                     place by the number of appended tokens
        c_t, k_rope: (batch, tokens, dc) and (batch, tokens, dR), one dtype;
                     k_rope un-rotated (keys are rotated by position inside
                     the attention)
        q_rope:      optional (batch * queries_per_seq, num_heads, dR) fp32,
                     rotated in place for the positions of the last
                     queries_per_seq appended tokens (needs rope_cos/sin)
        status:      optional int32 device tensor; element 0 is set to 1 when
                     a sequence has no room (that sequence is left unchanged)
        block_table, block_size: optional paged cache, as in ``mla_decode``
                     (capacity block_table.shape[1] * block_size per sequence)
    """
    _C = _load_ext()
    _C.append_kv_forward(kv_cache, seq_lens, c_t, k_rope, q_rope, rope_cos, rope_sin, seq_offsets, status,
                         *_cfg_args(cfg), block_table, block_size)


def absorb_q(q_nope: torch.Tensor, W_UK: torch.Tensor, cfg: "MLAConfig") -> torch.Tensor:
    """q_absorbed[..., h, c] = sum_i q_nope[..., h, i] * W_UK[h*dn + i, c] (fp32)."""
    _C = _load_ext()
    return _C.absorb_q_forward(q_nope, W_UK, *_cfg_args(cfg))


def mla_prefill(
    kv_cache: torch.Tensor,
    q_nope: torch.Tensor,
    q_rope: torch.Tensor,
    W_UK: torch.Tensor,
    W_UV: torch.Tensor,
    rope_cos: torch.Tensor,
    rope_sin: torch.Tensor,
    cfg: "MLAConfig",
    q_offsets: Optional[torch.Tensor] = None,
    seq_offsets: Optional[torch.Tensor] = None,
    seq_lens: Optional[torch.Tensor] = None,
    block_table: Optional[torch.Tensor] = None,
    block_size: int = 0,
    prefix_lens: Optional[torch.Tensor] = None,
    rotate_q: bool = False,
    max_seq_rows: int = 0,
    out_dtype: Optional[torch.dtype] = None,
    kernel_variant: int = 0,
) -> torch.Tensor:
    """Causal attention of several new tokens per sequence: whole prompts,
    pieces of them over what the cache holds already, drafted tokens.

    The new tokens' rows are in the cache (``append_kv``) and are each
    sequence's last: token j of n of a sequence with L rows is at position
    L - n + j and sees the rows up to its own.

    Args:
        kv_cache:    as in ``mla_decode``: (batch, capacity, dc + dR), packed
                     (rows, dc + dR) with ``seq_offsets``, or a paged pool with
                     ``block_table`` / ``block_size`` / ``seq_lens``
        q_nope:      (tokens, num_heads, qk_nope_head_dim) fp32 / fp16 / bf16,
                     the sequences' new tokens one after another
        q_rope:      (tokens, num_heads, qk_rope_head_dim), the same type; both
                     may be strided views whose last dimension is contiguous
                     (slices of one projection's output)
        q_offsets:   int32 (batch + 1,) device tensor starting at 0; sequence b
                     has tokens [q_offsets[b], q_offsets[b+1]); None: tokens /
                     batch each. Tokens behind the last sequence get zeros.
        prefix_lens: optional int32 (batch,) device tensor: the first
                     prefix_lens[b] rows of sequence b are seen by all of its
                     tokens (read in both directions)
        rotate_q:    q_rope is not rotated yet: rotated on the way by its
                     token's position (the tensor is left as it is)
        max_seq_rows: a region ends there (0: its capacity); bounds the
                     workspace of caches whose capacity is far beyond the
                     lengths
        out_dtype:   fp32 / fp16 / bf16; None: the queries' type
        kernel_variant: 0 = automatic, 1 = plain kernel, 2 = keys and values
                     expanded, 3 = queries absorbed

    Returns:
        (tokens, num_heads, v_head_dim) in out_dtype
    """
    _C = _load_ext()
    return _C.mla_prefill_forward(kv_cache, q_nope, q_rope, W_UK, W_UV, rope_cos, rope_sin, q_offsets, seq_offsets,
                                  *_cfg_args(cfg), seq_lens, block_table, block_size, prefix_lens, rotate_q,
                                  max_seq_rows, q_nope.dtype if out_dtype is None else out_dtype, kernel_variant)


@dataclass(frozen=True)
class SharedPrefix:
    """A prefix for ``mla_decode_shared``: its latent rows and, from
    ``expand_prefix``, their per-head keys and values. ``expanded`` belongs to
    the weights and tables that it was made with."""

    rows: torch.Tensor  # (prefix, kv_lora_rank + qk_rope_head_dim)
    expanded: torch.Tensor  # fp16 (fp16 rows) or bf16, the library's order
    num_heads: int

    @property
    def _tiles(self) -> int:
        return -(-self.rows.size(0) // 64)

    @property
    def k_nope(self) -> torch.Tensor:
        """Keys W_UK c_t as a view (tile, 2, 32, head, 8, 2, 2, 4): rows (zeros
        past the last), head, dims in order; ``reshape(-1, heads, 128)`` copies
        them into rows."""
        t, h = self._tiles, self.num_heads
        return self.expanded[:h * t * 8192].view(h, t, 2, 8, 2, 32, 2, 4).permute(1, 2, 5, 0, 3, 6, 4, 7)

    @property
    def v(self) -> torch.Tensor:
        """Values W_UV c_t as a view (tile, 4, 2, 2, 4, head, 4, 32)."""
        t, h = self._tiles, self.num_heads
        return self.expanded[h * t * 8192:2 * h * t * 8192].view(h, t, 4, 4, 2, 32, 2, 4).permute(1, 3, 6, 4, 7, 0, 2, 5)

    @property
    def k_rope(self) -> torch.Tensor:
        """Rotated rope keys as a view (tile, 2, 32, 4, 2, 2, 4)."""
        t, h = self._tiles, self.num_heads
        return self.expanded[2 * h * t * 8192:].view(t, 2, 4, 2, 32, 2, 4).permute(0, 1, 4, 2, 5, 3, 6)


def expand_prefix(
    kv_cache: torch.Tensor,
    W_UK: torch.Tensor,
    W_UV: torch.Tensor,
    rope_cos: torch.Tensor,
    rope_sin: torch.Tensor,
    cfg: "MLAConfig",
) -> SharedPrefix:
    """Expands a prefix's latent rows (prefix, dc + dR; fp16, bf16 or FP8) into
    per-head keys and values, once for the many steps that read them: 512 bytes
    per row and head, with which ``mla_decode_shared`` does under a third of
    the products for a large batch. kv_lora_rank 512, 128-dim heads, rope 64."""
    _C = _load_ext()
    return SharedPrefix(kv_cache, _C.expand_prefix_forward(kv_cache, W_UK, W_UV, rope_cos, rope_sin, *_cfg_args(cfg)),
                        cfg.num_heads)


def mla_decode_shared(
    prefix: Union[SharedPrefix, torch.Tensor],
    kv_cache: torch.Tensor,
    q_nope: torch.Tensor,
    q_rope: torch.Tensor,
    W_UK: torch.Tensor,
    W_UV: torch.Tensor,
    rope_cos: torch.Tensor,
    rope_sin: torch.Tensor,
    cfg: "MLAConfig",
    seq_offsets: Optional[torch.Tensor] = None,
    seq_lens: Optional[torch.Tensor] = None,
    block_table: Optional[torch.Tensor] = None,
    block_size: int = 0,
    out_dtype: torch.dtype = torch.float32,
    kernel_variant: int = 0,
) -> torch.Tensor:
    """``mla_decode`` for sequences that share a prefix, which is attended once
    for all of them.

    Args:
        prefix:      (prefix, dc + dR) latent rows at positions 0, 1, ..., in
                     kv_cache's type, or a ``SharedPrefix`` of them
        kv_cache, seq_offsets, seq_lens, block_table, block_size: the
                     sequences' own rows, as in ``mla_decode``; row i of a
                     sequence is at position prefix + i, and it may have none
        q_nope, q_rope, W_UK, W_UV: as in ``mla_decode``
        rope_cos / rope_sin: (>= prefix + longest sequence, dR / 2)
        out_dtype:   fp32 / fp16 / bf16
        kernel_variant: 0 = automatic, 1 = the prefix's latent rows, 2 = its
                     expanded form

    Returns:
        (batch, num_heads, v_head_dim) in out_dtype
    """
    _C = _load_ext()
    expanded = None
    if isinstance(prefix, SharedPrefix):
        if prefix.num_heads != cfg.num_heads:
            raise ValueError(f"prefix was expanded for {prefix.num_heads} heads, not {cfg.num_heads}")
        prefix, expanded = prefix.rows, prefix.expanded
    return _C.mla_decode_shared_forward(prefix, expanded, kv_cache, q_nope, q_rope, W_UK, W_UV, rope_cos, rope_sin,
                                        seq_offsets, *_cfg_args(cfg), seq_lens, block_table, block_size, out_dtype,
                                        kernel_variant)
