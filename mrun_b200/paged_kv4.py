"""A block-paged KV cache that holds keys and values in 4 bits, and the operators of a serving
step over it:

* ``kv_plan_step`` / ``kv_release`` -- pages, block tables and slot maps from request lengths, on
  the GPU (no host list, so a captured step can grow its own sequences)
* ``rope_kv4_append``  -- rotary positions (half or interleaved pairs, all or part of the head,
  scaled tables) and the 4-bit append of keys and values
* ``kv4_read``         -- what cached slots stand for, in bf16 or fp32
* ``kv4_paged_attention``   -- one query token per row over the cache
* ``kv4_prefill_attention`` -- causal attention of ragged query blocks over the cache

A pool is uint8 ``[pages, kv_heads, page_size / 16, block_bytes]``; a block is 16 tokens of one KV
head, contiguous: K codes ``[16, D / 2]`` (low nibble: the even dimension), V codes alike, then
``[16, D / group]`` pairs (scale, minimum) of bf16 for K and the same for V. ``group`` dimensions x
of a token are held as m = bf16(min x), s = bf16((max x - m) / 15) and codes round((x - m) / s),
and stand for m + s * code. At head_dim 128 a token of one head takes 136 bytes in one group and
160 in groups of 32, against 512 in bf16 (``paged_kv.PagedKVCache``, whose page-table conventions
this cache follows).
"""
from __future__ import annotations

import math
from functools import lru_cache
from typing import NamedTuple

import torch

from . import _lib

TILE = 16

KV_BAD_REQUEST = 1
KV_TABLE_FULL = 2
KV_TOKENS_FULL = 4
KV_POOL_EMPTY = 8
KV_BAD_SLOT = 16
KV_UNMAPPED = 32
KV_TIMEOUT = 64
KV_TOO_LONG = 128

_ERRORS = {
    KV_BAD_REQUEST: "a sequence out of range or twice in a step, a negative count, or a damaged page list",
    KV_TABLE_FULL: "a sequence grew past its block-table row",
    KV_TOKENS_FULL: "a step had more new tokens than max_tokens",
    KV_POOL_EMPTY: "the paged KV pool is exhausted",
    KV_BAD_SLOT: "an append saw a slot or position out of range",
    KV_UNMAPPED: "attention met an unmapped page",
    KV_TIMEOUT: "a wait inside an attention kernel ran out, its outputs are void",
    KV_TOO_LONG: "attention met a row longer than max_total_tokens or than its block-table row",
}


def kv4_block_bytes(head_dim: int, group: int) -> int:
    """Bytes of 16 tokens of one KV head."""
    if head_dim not in (64, 128) or group not in (32, 64, 128) or group > head_dim:
        raise ValueError("4-bit caches hold head_dim 64 or 128 in groups of 32, 64 or 128 dimensions, "
                         f"not {head_dim} in groups of {group}")
    return TILE * head_dim + 2 * TILE * (head_dim // group) * 4


def scaled_rope_tables(rotary_dim: int, theta: float, length: int, device: torch.device, *,
                       scaling: dict | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """cos/sin fp32 [length, rotary_dim/2] of a rotation that may be stretched for long contexts,
    evaluated in fp64. ``scaling`` (Hugging Face ``rope_scaling`` keys; None: plain) is one of

    * ``{"rope_type": "linear", "factor"}``: positions divided by the factor
    * ``{"rope_type": "ntk", "factor"}``: theta raised to theta * factor^(R / (R - 2))
    * ``{"rope_type": "llama3", "factor", "low_freq_factor", "high_freq_factor",
      "original_max_position_embeddings"}``: long wavelengths divided by the factor, short ones
      kept, a linear blend between
    * ``{"rope_type": "yarn", "factor", "original_max_position_embeddings", "beta_fast",
      "beta_slow", "truncate", "attention_factor", "mscale", "mscale_all_dim"}``: the same with a ramp
      over the dimensions (between whole ones unless ``truncate`` is false), and both tables times the
      attention factor: by default 0.1 ln(factor) + 1, or with both ``mscale`` numbers
      (0.1 mscale ln(factor) + 1) / (0.1 mscale_all_dim ln(factor) + 1)
    """
    if rotary_dim < 8 or rotary_dim % 8:
        raise ValueError("rotary_dim must be a positive multiple of 8")
    half = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim
    kind = "default" if scaling is None else scaling.get("rope_type", scaling.get("type", "default"))
    needs = {"default": (), "linear": ("factor",), "ntk": ("factor",),
             "llama3": ("factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"),
             "yarn": ("factor", "original_max_position_embeddings")}
    if kind not in needs:
        raise ValueError(f"unknown rotary scaling {kind!r}")
    missing = [key for key in needs[kind] if scaling.get(key) is None] if needs[kind] else []
    if missing:
        raise ValueError(f"{kind} rotary scaling needs {', '.join(missing)}")
    factor = 1.0 if kind == "default" else float(scaling["factor"])
    if not math.isfinite(factor) or factor < 1.0:
        raise ValueError("a rotary scaling factor must be at least 1")
    mult = 1.0
    if kind == "ntk":
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    inv = theta ** -half
    if kind == "linear":
        inv = inv / factor
    elif kind == "llama3":
        span = float(scaling["original_max_position_embeddings"])
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        turns = span * inv / (2 * math.pi)  # turns over the original context
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        inv = inv * keep + inv / factor * (1 - keep)
    elif kind == "yarn":
        span = float(scaling["original_max_position_embeddings"])

        def dim_of(turns: float) -> float:
            return rotary_dim * math.log(span / (turns * 2 * math.pi)) / (2 * math.log(theta))

        first, last = dim_of(float(scaling.get("beta_fast") or 32)), dim_of(float(scaling.get("beta_slow") or 1))
        if scaling.get("truncate", True):
            first, last = math.floor(first), math.ceil(last)
        first, last = max(first, 0), min(last, rotary_dim - 1)
        index = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
        keep = 1 - ((index - first) / max(last - first, 1e-3)).clamp(0, 1)
        inv = inv * keep + inv / factor * (1 - keep)

        def magnitude(m: float) -> float:
            return 0.1 * m * math.log(factor) + 1.0

        mult = scaling.get("attention_factor")
        if mult is None and scaling.get("mscale") and scaling.get("mscale_all_dim"):
            mult = magnitude(float(scaling["mscale"])) / magnitude(float(scaling["mscale_all_dim"]))
        mult = magnitude(1.0) if mult is None else float(mult)
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * inv
    return (angle.cos() * mult).float().contiguous(), (angle.sin() * mult).float().contiguous()


# ------------------------------------------------------------------ operators


class KVStepPlan(NamedTuple):
    """One step's page plan (device int32 tensors)."""

    q_starts: torch.Tensor  # [rows + 1] new tokens before each request
    row_len: torch.Tensor  # [rows] tokens of each request's sequence after the step
    positions: torch.Tensor  # [max_tokens] position of each new token in its sequence
    token_rows: torch.Tensor  # [max_tokens] its sequence
    slots: torch.Tensor  # [max_tokens] its cache slot, page * page_size + place in the page (-1: none)

    @classmethod
    def empty(cls, rows: int, max_tokens: int, device: torch.device) -> "KVStepPlan":
        pad = -max_tokens % 4  # the token lists are 16-byte aligned
        one = torch.empty(3 * (max_tokens + pad) + 2 * rows + 1, dtype=torch.int32, device=device)
        if pad:
            positions, _, token_rows, _, slots, _, q_starts, row_len = one.split_with_sizes(
                (max_tokens, pad, max_tokens, pad, max_tokens, pad, rows + 1, rows))
        else:
            positions, token_rows, slots, q_starts, row_len = one.split_with_sizes(
                (max_tokens, max_tokens, max_tokens, rows + 1, rows))
        return cls(q_starts, row_len, positions, token_rows, slots)


def kv_plan_step(
    new_tokens: torch.Tensor,
    lengths: torch.Tensor,
    block_table: torch.Tensor,
    free_pages: torch.Tensor,
    free_count: torch.Tensor,
    *,
    page_size: int,
    max_tokens: int,
    row_seq: torch.Tensor | None = None,
    lengths_out: torch.Tensor | None = None,
    free_count_out: torch.Tensor | None = None,
    error_flag: torch.Tensor | None = None,
    out: KVStepPlan | None = None,
) -> KVStepPlan:
    """Plan one step: request r appends ``new_tokens[r]`` tokens to sequence ``row_seq[r]`` (default
    r; distinct), whose committed tokens are ``lengths[seq]``. Takes the fresh pages from the stack
    ``free_pages[:free_count]`` and writes their ``block_table`` entries. ``lengths_out`` and
    ``free_count_out`` default to their inputs (updated in place). A step that does not fit changes
    nothing, gives every token slot -1 and sets ``error_flag`` bits (``KV_*``)."""
    device = _lib.require_cuda(new_tokens, lengths, block_table, free_pages, free_count, what="KV step plan")
    if out is None:
        out = KVStepPlan.empty(new_tokens.numel(), int(max_tokens), device)
    elif out.slots.numel() != max_tokens:
        raise ValueError(f"the plan holds {out.slots.numel()} tokens, not max_tokens={max_tokens}")
    _lib.ops().kv_plan_step(new_tokens, row_seq, lengths, lengths if lengths_out is None else lengths_out, block_table,
                            free_pages, free_count, free_count if free_count_out is None else free_count_out,
                            page_size, *out, error_flag)
    return out


def kv_release(seqs: torch.Tensor, lengths: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
               free_count: torch.Tensor, *, page_size: int, error_flag: torch.Tensor | None = None) -> None:
    """End the sequences ``seqs`` (int32): their pages return to the free stack in order, their
    block-table rows become -1 and their lengths 0."""
    _lib.require_cuda(seqs, lengths, block_table, free_pages, free_count, what="KV release")
    _lib.ops().kv_release(seqs, lengths, block_table, free_pages, free_count, page_size, error_flag)


def rope_kv4_append(
    k_in: torch.Tensor,
    v_in: torch.Tensor,
    pool: torch.Tensor,
    *,
    group: int,
    head_dim: int,
    slots: torch.Tensor,
    positions: torch.Tensor | None = None,
    q_in: torch.Tensor | None = None,
    num_heads: int = 0,
    rope: tuple[torch.Tensor, torch.Tensor] | None = None,
    interleaved: bool = False,
    qk_norm: tuple[torch.Tensor, torch.Tensor] | None = None,
    norm_eps: float = 1e-6,
    q_out: torch.Tensor | None = None,
    error_flag: torch.Tensor | None = None,
) -> torch.Tensor | None:
    """Rotate queries and keys and write keys and values to their slots in 4 bits.

    ``k_in`` / ``v_in``: bf16 rows [tokens, kv_heads * head_dim], ``q_in``: [tokens, num_heads *
    head_dim], each with a row stride of its own (slices of one fused projection output are fine).
    ``rope`` = (cos, sin) fp32 [positions, rotary_dim / 2]: the first rotary_dim dimensions of each head turn, in pairs
    (d, d + rotary_dim / 2) or, ``interleaved``, (2i, 2i + 1). ``qk_norm`` = (q weight, k weight):
    per-head RMSNorm before the rotation. A token with slot -1 is rotated but not stored. Returns
    the rotated queries, bf16 [tokens, num_heads, head_dim] (None without ``q_in``)."""
    device = _lib.require_cuda(k_in, v_in, pool, slots, positions, q_in, what="4-bit KV append")
    if pool.shape[-1] != kv4_block_bytes(head_dim, group):
        raise ValueError(f"the pool's blocks of {pool.shape[-1]} bytes do not hold head_dim {head_dim} "
                         f"in groups of {group}")
    if q_in is not None:
        if q_in.ndim != 2 or q_in.shape[1] != num_heads * head_dim:
            raise ValueError(f"q_in must be [tokens, num_heads * head_dim], got {tuple(q_in.shape)}")
        if q_out is None:
            q_out = torch.empty(q_in.shape[0], num_heads, head_dim, dtype=torch.bfloat16, device=device)
    cos, sin = rope if rope is not None else (None, None)
    qn, kn = qk_norm if qk_norm is not None else (None, None)
    _lib.ops().rope_kv4_append(q_in, k_in, v_in, pool, group, slots, positions, cos, sin, interleaved, qn, kn,
                               norm_eps, q_out, error_flag)
    return q_out


def kv4_read(pool: torch.Tensor, slots: torch.Tensor, *, group: int, head_dim: int,
             dtype: torch.dtype = torch.bfloat16,
             error_flag: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that ``slots`` (int32) stand for: two tensors [tokens, kv_heads,
    head_dim] of ``dtype`` (bf16 or fp32; zeros for slot -1)."""
    device = _lib.require_cuda(pool, slots, what="4-bit KV read")
    if pool.ndim != 4 or pool.shape[3] != kv4_block_bytes(head_dim, group):
        raise ValueError(f"the pool's blocks do not hold head_dim {head_dim} in groups of {group}")
    if dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"cached values are read as bf16 or fp32, not {dtype}")
    shape = (slots.numel(), pool.shape[1], head_dim)
    k, v = torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device)
    _lib.ops().kv4_read(pool, group, slots, k, v, error_flag)
    return k, v


_WORKSPACE = _lib.StreamScratch()
_PREFILL_WORKSPACE = _lib.StreamScratch()
_COUNTER_BYTES = 8192  # MRB_KV4_COUNTER_BYTES: what has to be zero of a workspace


@lru_cache(maxsize=4096)
def kv4_paged_attention_workspace_bytes(rows: int, hq: int, hkv: int, head_dim: int, max_total_tokens: int) -> int:
    return int(_lib.load().mrb_kv4_paged_attention_workspace(rows, hq, hkv, head_dim, max_total_tokens))


def kv4_paged_attention(
    query: torch.Tensor,
    pool: torch.Tensor,
    *,
    group: int,
    block_table: torch.Tensor,
    row_len: torch.Tensor,
    max_total_tokens: int,
    row_seq: torch.Tensor | None = None,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
    error_flag: torch.Tensor | None = None,
) -> torch.Tensor:
    """One query token per row, [rows, hq, d] bf16, over tokens ``[0, row_len[r])`` of sequence
    ``row_seq[r]`` (default r). ``max_total_tokens`` bounds the lengths (``KV_TOO_LONG``
    is set where one is cut). Rows without tokens give
    zeros. The workspace, when given, must be zeroed once and serve one stream or one graph; by
    default calls take their stream's, and captured calls one of the graph's own."""
    device = _lib.require_cuda(query, pool, block_table, row_len, what="4-bit paged attention")
    if query.dtype != torch.bfloat16:
        raise TypeError("4-bit paged attention runs on bf16 queries")
    if query.ndim != 3 or pool.ndim != 4:
        raise ValueError("query must be [rows, heads, head_dim] and the pool [pages, kv_heads, tiles, block_bytes]")
    q = query.contiguous()
    if out is None:
        out = torch.empty_like(q)
    rows, hq, d = q.shape
    need = kv4_paged_attention_workspace_bytes(rows, hq, pool.shape[1], d, max_total_tokens)
    if workspace is None:
        workspace = _WORKSPACE.get(device, need, counters=_COUNTER_BYTES)
    elif workspace.numel() < need:
        raise ValueError(f"workspace too small: {workspace.numel()} < {need} bytes")
    _lib.ops().kv4_paged_attention(q, pool, group, block_table, row_len, row_seq,
                                   1.0 / math.sqrt(d) if scale is None else scale, max_total_tokens, out, workspace,
                                   error_flag)
    return out


@lru_cache
def kv4_prefill_attention_workspace_bytes(head_dim: int) -> int:
    return int(_lib.load().mrb_kv4_prefill_attention_workspace(head_dim))


def kv4_prefill_attention(
    query: torch.Tensor,
    pool: torch.Tensor,
    *,
    group: int,
    block_table: torch.Tensor,
    q_starts: torch.Tensor,
    row_len: torch.Tensor,
    row_seq: torch.Tensor | None = None,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
    error_flag: torch.Tensor | None = None,
) -> torch.Tensor:
    """Causal attention of ragged query blocks: ``query[q_starts[r]:q_starts[r + 1]]`` ([tokens, hq,
    d] bf16) are the last tokens of row r's ``row_len[r]`` cached ones (sequence ``row_seq[r]``,
    default r), each attending up to itself. Tokens of no block (from ``q_starts[rows]`` on: padding, or
    all of them after a plan that did not fit) give zeros; in a given ``out`` they stay as they are. The
    workspace is as that of ``kv4_paged_attention``."""
    device = _lib.require_cuda(query, pool, block_table, q_starts, row_len, what="4-bit prefill attention")
    if query.dtype != torch.bfloat16:
        raise TypeError("4-bit prefill attention runs on bf16 queries")
    if query.ndim != 3 or pool.ndim != 4:
        raise ValueError("query must be [tokens, heads, head_dim] and the pool [pages, kv_heads, tiles, block_bytes]")
    q = query.contiguous()
    zero_rest = out is None
    if out is None:
        out = torch.empty_like(q) if row_len.numel() else torch.zeros_like(q)
    need = kv4_prefill_attention_workspace_bytes(q.shape[2])
    if workspace is None:
        workspace = _PREFILL_WORKSPACE.get(device, need, counters=_COUNTER_BYTES)
        if workspace is None:  # the head_dim has no kernel: the operator says so
            workspace = torch.empty(0, dtype=torch.uint8, device=device)
    elif workspace.numel() < need:
        raise ValueError(f"workspace too small: {workspace.numel()} < {need} bytes")
    _lib.ops().kv4_prefill_attention(q, pool, group, block_table, q_starts, row_len, row_seq,
                                     1.0 / math.sqrt(q.shape[2]) if scale is None else scale, out, workspace,
                                     error_flag, zero_rest)
    return out


# ------------------------------------------------------------------ the cache


class PagedKV4Cache:
    """Per-layer 4-bit pools with one block table, its page allocator and lengths on the GPU."""

    def __init__(self, *, num_layers: int, num_pages: int, kv_heads: int, head_dim: int, max_seqs: int,
                 max_pages_per_seq: int, device: torch.device, page_size: int = TILE,
                 group: int | None = None) -> None:
        if page_size < TILE or page_size % TILE:
            raise ValueError("page_size must be a multiple of 16 tokens")
        self.num_layers, self.num_pages = int(num_layers), int(num_pages)
        self.kv_heads, self.head_dim = int(kv_heads), int(head_dim)
        self.group = int(group) if group is not None else self.head_dim
        self.page_size = int(page_size)
        self.max_seqs, self.max_pages_per_seq = int(max_seqs), int(max_pages_per_seq)
        self.device = device
        block = kv4_block_bytes(self.head_dim, self.group)
        shape = (self.num_layers, self.num_pages, self.kv_heads, self.page_size // TILE, block)
        self.pool = torch.zeros(shape, dtype=torch.uint8, device=device)
        i32 = {"dtype": torch.int32, "device": device}
        self.block_table = torch.full((self.max_seqs, self.max_pages_per_seq), -1, **i32)
        self.lengths = torch.zeros(self.max_seqs, **i32)
        self.free_pages = torch.arange(self.num_pages - 1, -1, -1, **i32)  # pages are handed out from 0 on
        self.free_count = torch.full((1,), self.num_pages, **i32)
        self.error_flag = torch.zeros(1, **i32)

    @property
    def bytes_per_token(self) -> int:
        return self.num_layers * self.kv_heads * kv4_block_bytes(self.head_dim, self.group) // TILE

    def plan_step(self, new_tokens: torch.Tensor, *, max_tokens: int, row_seq: torch.Tensor | None = None,
                  out: KVStepPlan | None = None) -> KVStepPlan:
        """Map the pages of one step's new tokens and commit the new lengths (``kv_plan_step``)."""
        return kv_plan_step(new_tokens, self.lengths, self.block_table, self.free_pages, self.free_count,
                            page_size=self.page_size, max_tokens=max_tokens, row_seq=row_seq,
                            error_flag=self.error_flag, out=out)

    def release(self, seqs: torch.Tensor) -> None:
        """End sequences (device int32 ids); their pages are free for the next step."""
        kv_release(seqs, self.lengths, self.block_table, self.free_pages, self.free_count,
                   page_size=self.page_size, error_flag=self.error_flag)

    def append(self, layer: int, k_rows: torch.Tensor, v_rows: torch.Tensor, plan: KVStepPlan, *,
               q_rows: torch.Tensor | None = None, num_heads: int = 0, q_out: torch.Tensor | None = None,
               rope: tuple[torch.Tensor, torch.Tensor] | None = None, interleaved: bool = False,
               qk_norm: tuple[torch.Tensor, torch.Tensor] | None = None,
               norm_eps: float = 1e-6) -> torch.Tensor | None:
        return rope_kv4_append(k_rows, v_rows, self.pool[layer], group=self.group, head_dim=self.head_dim,
                               slots=plan.slots, positions=plan.positions, q_in=q_rows, num_heads=num_heads,
                               rope=rope, interleaved=interleaved, qk_norm=qk_norm, norm_eps=norm_eps, q_out=q_out,
                               error_flag=self.error_flag)

    def read(self, layer: int, slots: torch.Tensor, *,
             dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
        return kv4_read(self.pool[layer], slots, group=self.group, head_dim=self.head_dim, dtype=dtype,
                        error_flag=self.error_flag)

    def workspace_bytes(self, rows: int, num_heads: int, max_total_tokens: int) -> int:
        return kv4_paged_attention_workspace_bytes(rows, num_heads, self.kv_heads, self.head_dim, max_total_tokens)

    def prefill_workspace_bytes(self) -> int:
        return kv4_prefill_attention_workspace_bytes(self.head_dim)

    def attend(self, layer: int, query: torch.Tensor, row_len: torch.Tensor, *, max_total_tokens: int,
               row_seq: torch.Tensor | None = None, out: torch.Tensor | None = None,
               workspace: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
        return kv4_paged_attention(query, self.pool[layer], group=self.group, block_table=self.block_table,
                                   row_len=row_len, max_total_tokens=max_total_tokens, row_seq=row_seq, scale=scale,
                                   out=out, workspace=workspace, error_flag=self.error_flag)

    def attend_prefill(self, layer: int, query: torch.Tensor, plan: KVStepPlan, *,
                       row_seq: torch.Tensor | None = None, scale: float | None = None,
                       out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
        return kv4_prefill_attention(query, self.pool[layer], group=self.group, block_table=self.block_table,
                                     q_starts=plan.q_starts, row_len=plan.row_len, row_seq=row_seq, scale=scale,
                                     out=out, workspace=workspace, error_flag=self.error_flag)

    def check_errors(self) -> None:
        """Raise on what the steps since the last call reported (synchronises)."""
        bits = int(self.error_flag.item())
        if bits:
            self.error_flag.zero_()
            text = "; ".join(message for bit, message in _ERRORS.items() if bits & bit)
            if bits & KV_POOL_EMPTY:
                raise MemoryError(text)
            if bits & (KV_TABLE_FULL | KV_TOKENS_FULL | KV_TOO_LONG):
                raise OverflowError(text)
            raise RuntimeError(text)


__all__ = [
    "KVStepPlan",
    "PagedKV4Cache",
    "kv4_block_bytes",
    "kv4_paged_attention",
    "kv4_paged_attention_workspace_bytes",
    "kv4_prefill_attention",
    "kv4_prefill_attention_workspace_bytes",
    "kv4_read",
    "kv_plan_step",
    "kv_release",
    "rope_kv4_append",
    "scaled_rope_tables",
]
