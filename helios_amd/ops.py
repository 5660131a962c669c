"""Python call surface of the MI355X paged-KV hot path.

``varlen_attn`` keeps the keyword surface the reference uses at
src/helios/runtime/qwen3/paged_cache.py:316-329 and :506-519
(torch 2.13 ``torch.nn.attention.varlen.varlen_attn`` with ``block_table=``), so
that module can import it in place of torch's. ``kv_append``, ``kv_copy_pages`` and
``kv_gather`` replace ``PagedBatchCache._write`` (paged_cache.py:335-345),
``KVCache.restore_blocks``' copy (cache.py:131-147) and ``_gather_cpu``
(paged_cache.py:405-414).

Every function validates its arguments on the host (ValueError, like
``_validate_attention_inputs`` at paged_cache.py:352-375), allocates outputs and
workspaces with ``torch.empty`` on the query's device (the caching allocator owns
them), and launches on ``torch.cuda.current_stream()`` without synchronising.
"""

from __future__ import annotations

import ctypes
import math
import os
from collections.abc import Sequence
from typing import NamedTuple

import torch

from helios_amd import _capi

_SUPPORTED = {torch.bfloat16: _capi.HX_DTYPE_BF16, torch.float16: _capi.HX_DTYPE_FP16}

# With HELIOS_AMD_CHECK_ERRORS=1 every attention run synchronises and raises RuntimeError
# when the kernels flagged bad metadata (a page id outside the pool, a length clamped to
# max_k / max_q / the table width, a malformed cu_seq_q, or a plan / run mismatch). Off by
# default: reading the flag is a device-to-host round trip per call, and the reference's
# hot path never synchronises (tests/test_continuous_batching.py:499-518). The kernels
# never read or write out of bounds either way.
CHECK_ERRORS = os.environ.get("HELIOS_AMD_CHECK_ERRORS", "") not in ("", "0")

_WERR_TEXT = {
    _capi.HX_WERR_BAD_PAGE: "a block-table page id outside the pool",
    _capi.HX_WERR_CLAMPED_LEN: "a sequence length beyond max_k, max_q or the block table",
    _capi.HX_WERR_BAD_CU_SEQ: "cu_seq_q not monotone or beyond the query rows",
    _capi.HX_WERR_GRID: "more work items than the launch grid covered",
    _capi.HX_WERR_PLAN_MISMATCH: "a run whose shape differs from its plan",
    _capi.HX_WERR_BAD_QUERY_ROW: "a query row map entry outside the query tensor",
}


def describe_error_word(word: int) -> str:
    """Text for the HX_WERR_* bits of an attention workspace error word."""
    parts = [text for bit, text in _WERR_TEXT.items() if word & bit]
    return "; ".join(parts) if parts else "no error"


class MergeParts(NamedTuple):
    """A shared-prefix cascade merge for ``VarlenAttnPlan.run(..., merge=...)``: member k
    is the decode row of sequence ``member_seq[k]`` (``member_of_seq[b]``: sequence b's
    member index or -1); its parts are rows ``part_idx[part_start[k]:part_start[k + 1]]``
    of ``level_out`` ``[A, H, 128]`` with log-sum-exps ``level_lse`` ``[H, A]``. All on the
    device; the int arrays are contiguous int32.

    ``level_plan``: the plan that produces ``level_out`` / ``level_lse``, when its run so
    far covered only its decode and chunk phases (``phases=("decode", "chunk")``, same
    stream): the merging run then does that plan's combine phase too, in workgroups added
    to its own decode launch, instead of a launch of its own.

    ``level_block_table`` (and ``level_query_rows``, int64 rows of the merging run's
    query): the level plan has not run at all and holds no decode rows; the merging run
    (all three phases, no append) runs its chunk items too, in one chunk launch with its
    own, ahead of its decode launch. ``level_out`` / ``level_lse`` are then outputs of
    that run (any contents on entry)."""

    level_out: torch.Tensor
    level_lse: torch.Tensor
    member_seq: torch.Tensor
    member_of_seq: torch.Tensor
    part_start: torch.Tensor
    part_idx: torch.Tensor
    level_plan: "VarlenAttnPlan | None" = None
    level_block_table: torch.Tensor | None = None
    level_query_rows: torch.Tensor | None = None


class AuxRequest(NamedTuple):
    """Auxiliary outputs of varlen_attn (same field as torch's AuxRequest)."""

    lse: bool = False


def _stream_ptr(device: torch.device) -> int:
    """The current stream's handle on ``device`` (the raw lookup: no Stream object)."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    return torch._C._cuda_getCurrentRawStream(index)


def _require_gpu(*tensors: torch.Tensor) -> torch.device:
    device = tensors[0].device
    if device.type != "cuda":
        raise RuntimeError(
            "helios_amd kernels run on a ROCm device only; got tensors on "
            f"{device}. There is no CPU fallback."
        )
    for t in tensors[1:]:
        if t.device != device:
            raise ValueError("All tensors must be on the same device.")
    return device


def _elem_bytes(t: torch.Tensor) -> int:
    return t.element_size()


# --------------------------------------------------------------------- KV append
def kv_append(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    write_slots: torch.Tensor,
    keys: torch.Tensor,
    values: torch.Tensor,
) -> None:
    """``k_cache.view(-1, Hkv, d).index_copy_(0, write_slots, keys)``, same for V.

    ``k_cache``/``v_cache``: pool tensors whose trailing dims are ``[Hkv, d]`` and
    that are contiguous (``[num_pages, page_size, Hkv, d]`` in the reference).
    ``keys``/``values``: ``[T, Hkv, d]`` with a contiguous last dim (any row/head
    strides). ``write_slots``: int64 ``[T]`` flat slot ids (page * page_size + offset).
    """
    device = _require_gpu(k_cache, v_cache, write_slots, keys, values)
    _check_append(k_cache, v_cache, write_slots, keys, values)
    n_kv, head_dim = keys.shape[1], keys.shape[2]
    write_slots = write_slots.contiguous()
    pool_rows = k_cache.numel() // (n_kv * head_dim)
    code = _capi.lib().hx_kv_append(
        k_cache.data_ptr(), v_cache.data_ptr(), pool_rows,
        keys.data_ptr(), keys.stride(0), keys.stride(1),
        values.data_ptr(), values.stride(0), values.stride(1),
        write_slots.data_ptr(), keys.shape[0],
        n_kv, head_dim, _elem_bytes(keys),
        _stream_ptr(device),
    )
    _capi.check(code, "hx_kv_append")


def _check_append(k_cache, v_cache, write_slots, keys, values) -> None:
    """Argument checks shared by kv_append and the fused append path."""
    if k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype:
        raise ValueError("Key and value pools must have identical shapes and dtypes.")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("KV pools must be contiguous.")
    if keys.ndim != 3 or values.shape != keys.shape:
        raise ValueError("Appended keys and values must be [tokens, kv_heads, head_dim].")
    n_kv, head_dim = keys.shape[1], keys.shape[2]
    if tuple(k_cache.shape[-2:]) != (n_kv, head_dim):
        raise ValueError("Appended K/V heads do not match the pool layout.")
    if keys.dtype != k_cache.dtype or values.dtype != k_cache.dtype:
        raise ValueError("Appended K/V dtype must match the pool dtype.")
    if write_slots.dtype != torch.int64 or write_slots.ndim != 1 or write_slots.shape[0] != keys.shape[0]:
        raise ValueError("write_slots must be int64 [tokens].")
    if keys.stride(2) != 1 or values.stride(2) != 1:
        raise ValueError("Appended K/V must have a contiguous head_dim.")


# ----------------------------------------------------- q/k norm + RoPE + append
def qk_norm_rope_append(
    queries: torch.Tensor,
    keys: torch.Tensor,
    values: torch.Tensor,
    q_norm_weight: torch.Tensor,
    k_norm_weight: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    write_slots: torch.Tensor,
    eps: float,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """q_norm/k_norm + apply_rope of the new rows (layers.py:146-160) fused with the KV
    append (paged_cache.py:335-345).

    ``queries`` ``[T, Hq, 128]``, ``keys``/``values`` ``[T, Hkv, 128]`` (projection
    outputs; contiguous last dim, any row/head strides); ``q_norm_weight``/``k_norm_weight``
    fp32 ``[128]``; ``cos``/``sin`` fp32 ``[rope_rows, 128]``; ``positions`` int64 ``[T]``
    (flattened, e.g. ``PackedBatchCache.positions[0]``). Returns the normalised, rotated
    queries ``[T, Hq, 128]`` (``out`` if given); rotated keys and raw values land in the
    pools at ``write_slots``.
    """
    device = _require_gpu(queries, keys, values, q_norm_weight, k_norm_weight, cos, sin,
                          positions, k_cache, v_cache, write_slots)
    _check_append(k_cache, v_cache, write_slots, keys, values)
    if queries.ndim != 3 or queries.shape[0] != keys.shape[0] or queries.shape[2] != keys.shape[2]:
        raise ValueError("queries must be [tokens, q_heads, head_dim] matching the keys.")
    if queries.dtype != keys.dtype or queries.stride(2) != 1:
        raise ValueError("queries must share the K/V dtype and have a contiguous head_dim.")
    head_dim = queries.shape[2]
    _check_rope(q_norm_weight, k_norm_weight, cos, sin, head_dim)
    positions = positions.reshape(-1)
    if positions.dtype != torch.int64 or positions.numel() != queries.shape[0]:
        raise ValueError("positions must be int64 with one entry per row.")
    positions = positions.contiguous()
    if out is None:
        out = torch.empty(queries.shape, dtype=queries.dtype, device=device)
    elif out.shape != queries.shape or out.dtype != queries.dtype or out.stride(2) != 1:
        raise ValueError("out must match the queries' shape and dtype.")
    dtype = {torch.bfloat16: _capi.HX_DTYPE_BF16, torch.float16: _capi.HX_DTYPE_FP16}.get(queries.dtype)
    if dtype is None:
        raise ValueError("q/k/v must be bfloat16 or float16.")
    pool_rows = k_cache.numel() // (keys.shape[1] * head_dim)
    code = _capi.lib().hx_qk_norm_rope_append(
        queries.data_ptr(), queries.stride(0), queries.stride(1),
        keys.data_ptr(), keys.stride(0), keys.stride(1),
        values.data_ptr(), values.stride(0), values.stride(1),
        q_norm_weight.data_ptr(), k_norm_weight.data_ptr(),
        cos.data_ptr(), sin.data_ptr(), cos.shape[0],
        positions.data_ptr(), queries.shape[0],
        queries.shape[1], keys.shape[1], head_dim, float(eps), dtype,
        out.data_ptr(), out.stride(0), out.stride(1),
        k_cache.data_ptr(), v_cache.data_ptr(), pool_rows, write_slots.contiguous().data_ptr(),
        _stream_ptr(device),
    )
    _capi.check(code, "hx_qk_norm_rope_append")
    return out


def _check_rope(q_norm_weight, k_norm_weight, cos, sin, head_dim: int) -> None:
    """Checks of the norm weights and RoPE tables."""
    for name, w in (("q_norm_weight", q_norm_weight), ("k_norm_weight", k_norm_weight)):
        if w.dtype != torch.float32 or w.numel() != head_dim or not w.is_contiguous():
            raise ValueError(f"{name} must be a contiguous float32 [head_dim] tensor.")
    if (cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.shape != sin.shape
            or cos.ndim != 2 or cos.shape[1] != head_dim or not cos.is_contiguous()
            or not sin.is_contiguous()):
        raise ValueError("cos/sin must be contiguous float32 [rows, head_dim] tables.")


def qk_norm_rope_append_packed(
    queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, n_q_heads: int, q_norm_weight: torch.Tensor,
    k_norm_weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
    k_cache: torch.Tensor, v_cache: torch.Tensor, write_slots: torch.Tensor, eps: float,
) -> torch.Tensor | None:
    """``qk_norm_rope_append`` for projections as they come, queries ``[1, T, Hq * d]`` and
    keys / values ``[1, T, Hkv * d]`` (any row stride, contiguous heads), contiguous pools
    and index vectors, without making row views on the way: the same launch. None, and
    nothing launched, for any other layout, type or device."""
    dtype, index = queries.dtype, queries.get_device()
    code = _SUPPORTED.get(dtype)
    if code is None or index < 0 or queries.ndim != 3 or keys.ndim != 3 or k_cache.ndim != 4:
        return None
    one, rows, width = queries.shape
    n_kv, head_dim = k_cache.shape[2], k_cache.shape[3]
    if (one != 1 or width != n_q_heads * head_dim or keys.shape != (1, rows, n_kv * head_dim)
            or values.shape != keys.shape or keys.dtype is not dtype or values.dtype is not dtype
            or queries.stride(2) != 1 or keys.stride(2) != 1 or values.stride(2) != 1
            or k_cache.dtype is not dtype or v_cache.dtype is not dtype or v_cache.shape != k_cache.shape
            or not k_cache.is_contiguous() or not v_cache.is_contiguous()
            or write_slots.dtype is not torch.int64 or write_slots.ndim != 1 or write_slots.numel() != rows
            or positions.dtype is not torch.int64 or positions.ndim != 1 or positions.numel() != rows
            or not write_slots.is_contiguous() or not positions.is_contiguous()):
        return None
    for t in (keys, values, q_norm_weight, k_norm_weight, cos, sin, positions, k_cache, v_cache, write_slots):
        if t.get_device() != index:
            return None
    _check_rope(q_norm_weight, k_norm_weight, cos, sin, head_dim)
    out = torch.empty((rows, n_q_heads, head_dim), dtype=dtype, device=queries.device)
    status = _capi.lib().hx_qk_norm_rope_append(
        queries.data_ptr(), queries.stride(1), head_dim, keys.data_ptr(), keys.stride(1), head_dim,
        values.data_ptr(), values.stride(1), head_dim, q_norm_weight.data_ptr(), k_norm_weight.data_ptr(),
        cos.data_ptr(), sin.data_ptr(), cos.shape[0], positions.data_ptr(), rows, n_q_heads, n_kv, head_dim, eps, code,
        out.data_ptr(), width, head_dim, k_cache.data_ptr(), v_cache.data_ptr(), k_cache.shape[0] * k_cache.shape[1],
        write_slots.data_ptr(), torch._C._cuda_getCurrentRawStream(index))
    _capi.check(status, "hx_qk_norm_rope_append")
    return out


# ------------------------------------------------------------ attention merge
def attn_merge(out: torch.Tensor, lse_out: torch.Tensor, o_a: torch.Tensor, lse_a: torch.Tensor,
               rows: torch.Tensor, parts: tuple[torch.Tensor, torch.Tensor] | None = None) -> None:
    """In place: merge attention results over disjoint key sets by log-sum-exp weights.

    Without ``parts``, ``(o_a[j], lse_a[:, j])`` merges into ``(out[rows[j]],
    lse_out[:, rows[j]])``. With ``parts = (part_start, part_idx)`` (int32 ``[n + 1]`` and
    ``[P]``), entry j merges the o_a rows ``part_idx[part_start[j]:part_start[j + 1]]``
    into ``out[rows[j]]`` in one pass. ``out`` ``[T, H, 128]`` and ``o_a`` ``[A, H, 128]``
    (contiguous last dim), ``lse_out`` fp32 ``[H, T]``, ``lse_a`` fp32 ``[H, A]``
    contiguous, ``rows`` int64 ``[n]`` without repeats. A part index outside ``[0, A)``
    is skipped."""
    device = _require_gpu(out, lse_out, o_a, lse_a, rows)
    if out.ndim != 3 or o_a.ndim != 3 or out.shape[1:] != o_a.shape[1:] or out.dtype != o_a.dtype:
        raise ValueError("out and o_a must be [rows, heads, head_dim] of one dtype.")
    if out.stride(2) != 1 or o_a.stride(2) != 1:
        raise ValueError("out and o_a need a contiguous head_dim.")
    n_a, heads = o_a.shape[0], o_a.shape[1]
    n = rows.numel()
    if lse_out.dtype != torch.float32 or tuple(lse_out.shape) != (heads, out.shape[0]) or not lse_out.is_contiguous():
        raise ValueError("lse_out must be contiguous float32 [heads, rows].")
    # The kernel bounds part indices by lse_a's row stride, so that stride must be o_a's
    # row count: lse_a contiguous [heads, n_a].
    if lse_a.dtype != torch.float32 or tuple(lse_a.shape) != (heads, n_a) or not lse_a.is_contiguous():
        raise ValueError("lse_a must be contiguous float32 [heads, rows].")
    if rows.dtype != torch.int64 or rows.ndim != 1 or not rows.is_contiguous():
        raise ValueError("rows must be contiguous int64 [n].")
    start_ptr = idx_ptr = None
    n_parts = 0
    if parts is None:
        if n != n_a:
            raise ValueError("without parts, rows must have one entry per o_a row.")
    else:
        part_start, part_idx = parts
        for name, t in (("part_start", part_start), ("part_idx", part_idx)):
            if t.dtype != torch.int32 or t.ndim != 1 or not t.is_contiguous() or t.device != device:
                raise ValueError(f"{name} must be a contiguous int32 vector on the device.")
        if part_start.numel() != n + 1:
            raise ValueError("part_start must have one entry per row plus one.")
        start_ptr, idx_ptr = part_start.data_ptr(), part_idx.data_ptr()
        n_parts = part_idx.numel()
    dtype = _SUPPORTED.get(out.dtype)
    if dtype is None:
        raise ValueError("attention outputs must be bfloat16 or float16.")
    code = _capi.lib().hx_attn_merge(
        out.data_ptr(), out.stride(0), out.stride(1), lse_out.data_ptr(), out.shape[0],
        o_a.data_ptr(), o_a.stride(0), o_a.stride(1), lse_a.data_ptr(), n_a,
        rows.data_ptr(), start_ptr, idx_ptr, n_parts, n, heads, o_a.shape[2], dtype, _stream_ptr(device),
    )
    _capi.check(code, "hx_attn_merge")


# ------------------------------------------------- between the block's products
def add_rms_norm(x: torch.Tensor, y: torch.Tensor | None, norm_weight: torch.Tensor,
                 eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """``(s, RMSNorm(s))`` of ``s = x + y`` (``s = x`` without ``y``): the residual add and
    the norm after it (layers.py:30-40, :202-232) in one launch. ``x`` / ``y`` bfloat16 or
    float16 ``[..., hidden]`` contiguous; ``norm_weight`` ``[hidden]``, float32 (another
    floating type is widened first)."""
    device = _require_gpu(x, norm_weight) if y is None else _require_gpu(x, norm_weight, y)
    dtype = _SUPPORTED.get(x.dtype)
    if dtype is None:
        raise ValueError("add_rms_norm supports bfloat16 and float16.")
    if not x.is_contiguous() or x.ndim < 1 or (y is not None and (y.shape != x.shape or y.dtype != x.dtype
                                                                 or not y.is_contiguous())):
        raise ValueError("x and y must be contiguous, of one shape and dtype.")
    hidden = x.shape[-1]
    if tuple(norm_weight.shape) != (hidden,) or not norm_weight.is_floating_point():
        raise ValueError("norm_weight must be floating-point [hidden].")
    norm_weight = norm_weight.float().contiguous()  # no copy for the usual float32 vector
    total = x if y is None else torch.empty_like(x)
    normed = torch.empty_like(x)
    if x.numel():
        code = _capi.lib().hx_add_rms_norm(
            x.data_ptr(), hidden, None if y is None else y.data_ptr(), hidden, norm_weight.data_ptr(), eps,
            x.numel() // hidden, hidden, dtype, None if y is None else total.data_ptr(), normed.data_ptr(),
            _stream_ptr(device))
        _capi.check(code, "hx_add_rms_norm")
    return total, normed


def swiglu(gate_up: torch.Tensor) -> torch.Tensor:
    """``silu(gate) * up`` (layers.py:13-27) of ``gate_up`` ``[..., 2 * ffn]`` (gate first),
    contiguous bfloat16 or float16; ``[..., ffn]``."""
    device = _require_gpu(gate_up)
    dtype = _SUPPORTED.get(gate_up.dtype)
    if dtype is None:
        raise ValueError("swiglu supports bfloat16 and float16.")
    if gate_up.ndim < 1 or gate_up.shape[-1] % 2 or not gate_up.is_contiguous():
        raise ValueError("gate_up must be contiguous [..., 2 * ffn].")
    ffn = gate_up.shape[-1] // 2
    out = torch.empty((*gate_up.shape[:-1], ffn), dtype=gate_up.dtype, device=device)
    if out.numel():
        code = _capi.lib().hx_swiglu(gate_up.data_ptr(), 2 * ffn, out.numel() // ffn, ffn, dtype, out.data_ptr(),
                                     _stream_ptr(device))
        _capi.check(code, "hx_swiglu")
    return out


def block_linear(x: torch.Tensor, weight: torch.Tensor, *, norm_weight: torch.Tensor | None = None,
                 eps: float = 0.0, residual: torch.Tensor | None = None, swiglu: bool = False) -> torch.Tensor:
    """``x @ weight.t()`` for ticks of up to 16 rows, with the decoder block's steps around it
    (layers.py:13-40, :202-232) in the same launch: ``x`` RMSNormed first with
    ``norm_weight``; ``residual`` added to the rounded product; ``swiglu``: ``weight`` holds
    gate, then up rows, and the result is ``silu(gate) * up``. Values round to the dtype where
    the separate steps round them. ``x`` ``[..., K]`` and ``residual`` ``[..., N]`` contiguous,
    ``weight`` ``[N, K]`` (``[2 N, K]``) contiguous, bfloat16 or float16, K a multiple of 64
    and N of 16."""
    device = x.device
    if device.type != "cuda" or weight.device != device:
        _require_gpu(x, weight)
    dtype = _SUPPORTED.get(x.dtype)
    if dtype is None or weight.dtype != x.dtype:
        raise ValueError("block_linear supports bfloat16 and float16 x and weight of one dtype.")
    k = x.shape[-1]
    if weight.ndim != 2 or weight.shape[1] != k or not weight.is_contiguous() or not x.is_contiguous():
        raise ValueError("x must be contiguous [..., K] and weight contiguous [N, K].")
    cols = weight.shape[0]
    if swiglu:
        if cols % 2 or residual is not None:
            raise ValueError("swiglu takes a weight of gate and up rows and no residual.")
        cols //= 2
    shape = (*x.shape[:-1], cols)
    if residual is not None and (residual.shape != shape or residual.dtype != x.dtype or residual.device != device
                                 or not residual.is_contiguous()):
        raise ValueError("residual must be contiguous, of the result's shape and dtype.")
    if norm_weight is not None:
        if tuple(norm_weight.shape) != (k,) or norm_weight.device != device or not norm_weight.is_floating_point():
            raise ValueError("norm_weight must be floating-point [K].")
        norm_weight = norm_weight.float().contiguous()  # no copy for the usual float32 vector
    if k == 0:  # sums of no terms
        zero = torch.zeros(shape, dtype=x.dtype, device=device)
        return zero if residual is None else residual + zero
    out = torch.empty(shape, dtype=x.dtype, device=device)
    code = _capi.lib().hx_skinny_gemm(
        x.data_ptr(), k, x.numel() // k, weight.data_ptr(), k, cols, k, dtype,
        None if norm_weight is None else norm_weight.data_ptr(), eps,
        None if residual is None else residual.data_ptr(), cols, 1 if swiglu else 0,
        out.data_ptr(), cols, _stream_ptr(device))
    _capi.check(code, "hx_skinny_gemm")
    return out


# ------------------------------------------- attention over selected blocks of the cache
MAX_SELECT_BLOCKS = 16384  # blocks of a sequence that select_blocks can order


def _pool_layout(name: str, pool: torch.Tensor) -> tuple[int, int, int, int, int]:
    """A pool's dtype code, pages, page size, KV heads and head dim, checked for the block operators."""
    shape = pool.shape
    if len(shape) != 4 or not pool.is_contiguous() or 0 in shape:
        raise ValueError(f"{name} must be a contiguous [pages, page_size, kv_heads, head_dim] pool.")
    dtype = _SUPPORTED.get(pool.dtype)
    if dtype is None:
        raise ValueError(f"{name} must be bfloat16 or float16.")
    pages, page_size, n_kv, head_dim = shape
    _check_head_dim(head_dim)
    return dtype, pages, page_size, n_kv, head_dim


def _check_head_dim(head_dim: int) -> None:
    if head_dim % 8 or head_dim > 256:
        raise ValueError("head_dim must be a multiple of 8 from 8 to 256.")


def _check_block_size(block_size: int, page_size: int) -> None:
    if not 16 <= block_size <= 1024 or block_size & (block_size - 1) or page_size % block_size:
        raise ValueError("block_size must be a power of two from 16 to 1024 that divides the page size.")


def _table_layout(block_table: torch.Tensor) -> tuple[int, int, int]:
    """A block table's rows, width and row stride, checked."""
    shape = block_table.shape
    if block_table.dtype == torch.int32 and len(shape) == 2 and shape[1] >= 1:
        batch, width = shape
        if block_table.is_contiguous():
            return batch, width, width
        row, entry = block_table.stride()
        if batch <= 1:
            row = width  # a single row's stride may be anything
        if (width == 1 or entry == 1) and row >= width:
            return batch, width, row
    raise ValueError("block_table must be int32 [batch, width] with contiguous rows.")


def _check_rows(queries: int, key_counts: torch.Tensor, rows: torch.Tensor | None, row_seq: torch.Tensor | None,
                batch: int, device: torch.device) -> int:
    """Checks of the query rows of a selection; their number."""
    n = key_counts.numel()
    for name, t, dtype in (("key_counts", key_counts, torch.int32), ("row_seq", row_seq, torch.int32),
                           ("rows", rows, torch.int64)):
        if t is not None and (t.dtype != dtype or t.shape != (n,) or not t.is_contiguous() or t.device != device):
            raise ValueError(f"{name} must be a contiguous {dtype} vector, one entry per query row, on the device.")
    if rows is None and n != queries:
        raise ValueError("without rows, key_counts must have one entry per query.")
    if row_seq is None and n > batch:
        raise ValueError("without row_seq, the block table must have a row per query row.")
    return n


def _vector_rows(query: torch.Tensor) -> torch.Tensor:
    """``query`` with heads that 16-byte loads may take: itself, or a contiguous copy."""
    row, head, element = query.stride()
    if element != 1 or row % 8 or head % 8 or query.data_ptr() % 16:
        return query.clone(memory_format=torch.contiguous_format)
    return query


def kv_block_bounds(k_cache: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor, cu_seq_q: torch.Tensor,
                    seqused_k: torch.Tensor, *, max_q: int) -> None:
    """Key bounds of the blocks that a tick's new tokens touched, in place, after those tokens
    are in the pool: ``bounds[page, block, h, 0] / [..., 1]`` is the elementwise lowest /
    highest key of head h among the block's tokens so far.

    ``k_cache`` ``[pages, page_size, kv_heads, head_dim]`` contiguous, bfloat16 or float16;
    ``bounds`` ``[pages, page_size // block_size, kv_heads, 2, head_dim]`` contiguous, of its
    dtype (a block is a power of two of 16 to 1024 tokens); ``block_table`` / ``cu_seq_q`` /
    ``seqused_k`` as for ``varlen_attn``. A block is read whole and its former bounds never,
    so a page that was reused or truncated needs no clearing. ``max_q`` is at least the longest
    sequence's new tokens. A NaN key makes both bounds NaN."""
    device = _require_gpu(k_cache, bounds, block_table, cu_seq_q, seqused_k)
    dtype, pages, page_size, n_kv, head_dim = _pool_layout("k_cache", k_cache)
    layout = bounds.shape
    if len(layout) != 5 or layout[1] < 1 or page_size % layout[1]:
        raise ValueError("bounds must be [pages, blocks per page, kv_heads, 2, head_dim].")
    block_size = page_size // layout[1]
    _check_block_size(block_size, page_size)
    if layout != (pages, layout[1], n_kv, 2, head_dim) or bounds.dtype != k_cache.dtype or not bounds.is_contiguous():
        raise ValueError("bounds must be contiguous [pages, blocks per page, kv_heads, 2, head_dim] of the pool's dtype.")
    batch = seqused_k.numel()
    for name, t, count in (("cu_seq_q", cu_seq_q, batch + 1), ("seqused_k", seqused_k, batch)):
        if t.dtype != torch.int32 or t.shape != (count,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 vector of {count} values.")
    table_rows, width, table_stride = _table_layout(block_table)
    if table_rows != batch:
        raise ValueError("block_table must have a row per sequence.")
    if max_q < 0:
        raise ValueError("max_q must be non-negative.")
    code = _launch(device, _capi.lib().hx_kv_block_bounds, k_cache.data_ptr(), bounds.data_ptr(), pages, page_size,
                   block_size, n_kv, head_dim, dtype, block_table.data_ptr(), table_stride, width,
                   cu_seq_q.data_ptr(), seqused_k.data_ptr(), batch, max_q)
    _capi.check(code, "hx_kv_block_bounds")


def select_blocks(query: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor, key_counts: torch.Tensor,
                  budget: int, *, block_size: int, sink: int = 1, recent: int = 2, row_seq: torch.Tensor | None = None,
                  rows: torch.Tensor | None = None) -> torch.Tensor:
    """The blocks each query row attends to, per KV head: int32 ``[n, kv_heads, budget]``,
    ascending, -1 behind a row's last.

    ``query`` ``[T, Hq, d]``; entry i of ``key_counts`` (int32 ``[n]``) is the number of keys
    that query row ``rows[i]`` (int64; None: i) sees of sequence ``row_seq[i]`` (int32; None:
    i), whose pages are ``block_table[row_seq[i]]``. The first ``sink`` and the last
    ``recent`` (at least 1) blocks are always among them; the others are those with the largest
    ``sum_g sum_d max(q_g[d] * lower[d], q_g[d] * upper[d])`` over the query heads g of the KV
    head, an upper bound of their summed scores, computed in 64 bits (equal ones: the
    earlier block; NaN: as infinity). A row with no more than ``budget`` blocks gets them all."""
    device = _require_gpu(query, bounds, block_table, key_counts)
    layout = query.shape
    if len(layout) != 3 or layout[2] < 1:
        raise ValueError("query must be [rows, n_q_heads, head_dim].")
    queries, n_q, head_dim = layout
    dtype = _SUPPORTED.get(query.dtype)
    if dtype is None or bounds.dtype != query.dtype:
        raise ValueError("query and bounds must be bfloat16 or float16, of one dtype.")
    layout = bounds.shape
    if len(layout) != 5 or layout[3] != 2 or layout[4] != head_dim or 0 in layout or not bounds.is_contiguous():
        raise ValueError("bounds must be contiguous [pages, blocks per page, kv_heads, 2, head_dim].")
    pages, per_page, n_kv = layout[:3]
    page_size = per_page * block_size
    _check_block_size(block_size, page_size)
    _check_head_dim(head_dim)
    if n_q < 1 or n_q % n_kv:
        raise ValueError(f"GQA needs n_q_heads ({n_q}) to be a multiple of n_kv_heads ({n_kv}).")
    batch, width, table_stride = _table_layout(block_table)
    if sink < 0 or recent < 1 or sink + recent > budget:
        raise ValueError("budget must cover sink (at least 0) and recent (at least 1) blocks.")
    if width * per_page > MAX_SELECT_BLOCKS:
        raise ValueError(f"a block table may cover at most {MAX_SELECT_BLOCKS} blocks; use larger ones.")
    n = _check_rows(queries, key_counts, rows, row_seq, batch, device)
    blocks = key_counts.new_empty((n, n_kv, budget))
    if n == 0:
        return blocks
    query = _vector_rows(query)
    lib = _capi.lib()
    ws_bytes = lib.hx_select_blocks_workspace_bytes(n, n_kv, width * per_page)
    workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
    q_row, q_head, _ = query.stride()
    code = _launch(
        device, lib.hx_select_blocks, query.data_ptr(), q_row, q_head, queries,
        None if rows is None else rows.data_ptr(), None if row_seq is None else row_seq.data_ptr(),
        key_counts.data_ptr(), n, n_q, n_kv, head_dim, dtype, bounds.data_ptr(), pages, page_size, block_size,
        block_table.data_ptr(), table_stride, batch, width, budget, sink, recent, blocks.data_ptr(),
        workspace.data_ptr(), ws_bytes)
    _capi.check(code, "hx_select_blocks")
    return blocks


def block_sparse_attn(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, blocks: torch.Tensor,
                      block_table: torch.Tensor, key_counts: torch.Tensor, *, block_size: int,
                      scale: float | None = None, row_seq: torch.Tensor | None = None,
                      rows: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of each query row over its listed blocks: ``softmax(scale * q . k) v`` over
    the keys of ``blocks[i, h // group]`` (int32 ``[n, kv_heads, budget]``, as ``select_blocks``
    gives them) below ``key_counts[i]``, in fp32, rounded once. Returns ``[T, Hq, d]`` like
    ``query``.

    ``rows`` / ``row_seq`` / ``key_counts`` / ``block_table`` as for ``select_blocks``; the
    pools ``[pages, page_size, kv_heads, head_dim]`` contiguous. Entries that are negative or
    past the keys are skipped, a block listed twice counts twice, a row without any key gets
    zeros. With ``rows`` (each at most once) only those rows of ``out`` are written: the
    others stay as they were (zeros when ``out`` is not given). Whatever the pool holds behind
    a sequence's last key is not read. An infinite or NaN element of a value that a row sees
    makes that element of its result infinite or NaN, at any weight. Of a key, a score of -inf
    is a weight of 0 (zeros for a row whose scores all are), one of +inf or NaN makes the row
    NaN, as in ``varlen_attn``."""
    device = _require_gpu(query, k_cache, v_cache, blocks, block_table, key_counts)
    dtype, pages, page_size, n_kv, head_dim = _pool_layout("k_cache", k_cache)
    _check_block_size(block_size, page_size)
    if v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype or not v_cache.is_contiguous():
        raise ValueError("Key and value pools must be contiguous, of one shape and dtype.")
    shape = query.shape
    if len(shape) != 3 or shape[2] != head_dim or query.dtype != k_cache.dtype:
        raise ValueError("query must be [rows, n_q_heads, head_dim] of the pools' dtype.")
    queries, n_q, _ = shape
    if n_q < 1 or n_q % n_kv:
        raise ValueError(f"GQA needs n_q_heads ({n_q}) to be a multiple of n_kv_heads ({n_kv}).")
    batch, width, table_stride = _table_layout(block_table)
    n = _check_rows(queries, key_counts, rows, row_seq, batch, device)
    listed = blocks.shape
    if blocks.dtype != torch.int32 or len(listed) != 3 or listed[0] != n or listed[1] != n_kv or listed[2] < 1 \
            or not blocks.is_contiguous():
        raise ValueError("blocks must be contiguous int32 [n, kv_heads, budget].")
    if out is None:
        out = (query.new_empty if rows is None else query.new_zeros)(shape)
    elif out.shape != shape or out.dtype != query.dtype or out.device != device or out.stride(2) != 1 \
            or out.data_ptr() % 4 or out.stride(0) % 2 or out.stride(1) % 2:
        raise ValueError("out must have the query's shape, dtype and device, a contiguous head_dim and even strides.")
    if n == 0:
        return out
    query = _vector_rows(query)
    scale = 1.0 / math.sqrt(head_dim) if scale is None else float(scale)
    budget, lib = listed[2], _capi.lib()
    ws_bytes = lib.hx_block_sparse_workspace_bytes(n, n_q, n_kv, head_dim, budget, block_size)
    workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes else None
    q_row, q_head, _ = query.stride()
    out_row, out_head, _ = out.stride()
    code = _launch(
        device, lib.hx_block_sparse_attn, query.data_ptr(), q_row, q_head, queries,
        None if rows is None else rows.data_ptr(), None if row_seq is None else row_seq.data_ptr(),
        key_counts.data_ptr(), n, k_cache.data_ptr(), v_cache.data_ptr(), pages, page_size, block_size,
        blocks.data_ptr(), budget, block_table.data_ptr(), table_stride, batch, width, n_q, n_kv, head_dim, scale,
        dtype, out.data_ptr(), out_row, out_head, None if workspace is None else workspace.data_ptr(), ws_bytes)
    _capi.check(code, "hx_block_sparse_attn")
    return out


# ------------------------------------------------------- products with 4-bit weights
class Int4Weight(NamedTuple):
    """A weight matrix ``[rows, k]`` in 4 bits with a scale and a zero point per ``group``
    elements of k: ``W[n, k] = scale[k // group, n] * (q[n, k] - zero[k // group, n])``.
    ``packed`` holds q and ``steps`` (int32) a scale's bits in the low half and those of 16 + a
    zero point in the high one, both in the order the kernel reads them (hx_int4_gemm);
    ``dtype`` is the scales' and the products' type. Made by ``int4_quantize`` or
    ``int4_pack``."""

    packed: torch.Tensor
    steps: torch.Tensor
    rows: int
    k: int
    group: int
    dtype: torch.dtype


def int4_pack(values: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor) -> Int4Weight:
    """``Int4Weight`` of integers 0..15 ``values`` ``[rows, k]`` (uint8), ``scales``
    ``[k / group, rows]`` (bfloat16 or float16) and ``zeros`` (uint8, 0..15) of the same
    shape; the group (32, 64 or 128) follows from the shapes. Done once per weight, in torch
    operations, on the tensors' device."""
    if values.ndim != 2 or values.dtype != torch.uint8 or min(values.shape) < 1:
        raise ValueError("values must be uint8 [rows, k].")
    rows, k = values.shape
    if scales.ndim != 2 or scales.shape[1] != rows or scales.dtype not in _SUPPORTED:
        raise ValueError("scales must be bfloat16 or float16 [k / group, rows].")
    if zeros.shape != scales.shape or zeros.dtype != torch.uint8:
        raise ValueError("zeros must be uint8, of the scales' shape.")
    if scales.device != values.device or zeros.device != values.device:
        raise ValueError("All tensors must be on the same device.")
    group = k // scales.shape[0] if scales.shape[0] else 0
    if group not in (32, 64, 128) or group * scales.shape[0] != k:
        raise ValueError(f"{k} elements in {scales.shape[0]} groups: a group is 32, 64 or 128 elements.")
    if int(values.max()) > 15 or int(zeros.max()) > 15:
        raise ValueError("values and zeros must lie in 0..15.")
    more_k, more_rows = -k % 128, -rows % 16
    q = torch.nn.functional.pad(values, (0, more_k, 0, more_rows)).to(torch.int64)
    q = q.view(-1, 16, q.shape[1] // 128, 4, 4, 8)  # tile, row, block, word, k group of a lane, element
    shift = torch.tensor([4 * (j // 2) + 16 * (j % 2) for j in range(8)], device=q.device)
    words = (q << shift).sum(dim=-1) << 3
    words = (words & 0xffffffff) | words >> 32  # turned by 3
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
    packed = words.permute(0, 2, 4, 1, 3).contiguous().view(torch.uint8)
    low, high = (t.contiguous().view(torch.int16).to(torch.int32) & 0xffff
                 for t in (scales, (zeros.to(torch.float32) + 16).to(scales.dtype)))
    steps = low | high << 16
    steps = torch.nn.functional.pad(steps, (0, more_rows, 0, more_k // group))
    steps = steps.view(-1, 128 // group, (rows + more_rows) // 16, 16).permute(2, 0, 3, 1).contiguous()
    return Int4Weight(packed.view(packed.shape[0], packed.shape[1], 64, 16), steps, rows, k, group, scales.dtype)


def int4_quantize(weight: torch.Tensor, group: int = 128) -> Int4Weight:
    """``weight`` ``[rows, k]`` (bfloat16 or float16) in 4 bits: per row and ``group`` (32, 64
    or 128) elements the 16 steps from the smallest (or 0) to the largest (or 0), each
    element to the nearest. Done once per weight, in torch operations."""
    if weight.ndim != 2 or weight.dtype not in _SUPPORTED or min(weight.shape) < 1:
        raise ValueError("weight must be bfloat16 or float16 [rows, k].")
    rows, k = weight.shape
    if group not in (32, 64, 128) or k % group:
        raise ValueError("group must be 32, 64 or 128 and divide k.")
    w = weight.float().view(rows, k // group, group) if weight.is_contiguous() else \
        weight.float().reshape(rows, k // group, group)
    if not bool(torch.isfinite(w).all()):
        raise ValueError("weight must be finite.")
    low, high = w.amin(dim=-1).clamp(max=0), w.amax(dim=-1).clamp(min=0)
    scale = (high / 15 - low / 15).to(weight.dtype)  # high - low may leave fp32
    step = scale.float().masked_fill(scale == 0, 1.0)[..., None]  # a group of zeros
    zero = (-low[..., None] / step).round().clamp(0, 15)
    values = ((w / step).round() + zero).clamp(0, 15).to(torch.uint8).view(rows, k)
    return int4_pack(values, scale.t().contiguous(), zero[..., 0].t().to(torch.uint8).contiguous())


def _check_int4(weight: Int4Weight, device: torch.device) -> int:
    """Checks of a packed weight; its dtype code."""
    packed, steps, rows, k, group, dtype = weight
    if group not in (32, 64, 128) or k % group or k < 1 or rows < 1:
        raise ValueError("the weight's group must be 32, 64 or 128 and divide its k.")
    blocks, tiles = -(-k // 128), -(-rows // 16)
    if packed.dtype != torch.uint8 or packed.shape != (tiles, blocks, 64, 16) or steps.dtype != torch.int32 \
            or steps.shape != (tiles, blocks, 16, 128 // group) or dtype not in _SUPPORTED:
        raise ValueError("an Int4Weight's tensors do not have the shapes and dtypes that int4_pack gives.")
    if packed.device != device or steps.device != device or not packed.is_contiguous() or not steps.is_contiguous():
        raise ValueError("an Int4Weight's tensors must be contiguous, on the product's device.")
    return _SUPPORTED[dtype]


def _launch(device: torch.device, fn, *args) -> int:
    """``fn(*args, stream)`` on ``device``'s current stream, with ``device`` the current one."""
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    if device.index == torch._C._cuda_getDevice():
        return fn(*args, stream)
    with torch.cuda.device(device):
        return fn(*args, stream)


INT4_MAX_ROWS = 64  # rows of x that one int4_linear takes


def int4_linear(x: torch.Tensor, weight: Int4Weight, *, norm_weight: torch.Tensor | None = None, eps: float = 0.0,
                residual: torch.Tensor | None = None, swiglu: bool = False) -> torch.Tensor:
    """``block_linear`` with 4-bit weights, for up to 64 rows: ``x @ W.t()`` with ``x``
    RMSNormed first by ``norm_weight``, ``residual`` added, or, with ``swiglu`` (``W`` holds
    gate, then up rows), ``silu(gate) * up``, in one launch. In fp32 and rounded once, at the
    end. ``x`` ``[..., k]`` and ``residual`` ``[..., n]`` contiguous, in the weight's dtype, ``x``
    16-byte aligned. More rows: ``int4_dequantize``, which rounds W to its type, and a library
    product."""
    device = _require_gpu(x)
    dtype = _check_int4(weight, device)
    cols, k = weight.rows, weight.k
    shape = x.shape
    if len(shape) < 1 or x.dtype != weight.dtype or shape[-1] != k or not x.is_contiguous():
        raise ValueError("x must be contiguous [..., k], in the weight's dtype.")
    if swiglu:
        if cols % 2 or residual is not None:
            raise ValueError("swiglu takes a weight of gate and up rows and no residual.")
        cols //= 2
    shape = (*shape[:-1], cols)
    if residual is not None and (residual.shape != shape or residual.dtype != x.dtype or residual.device != device
                                 or not residual.is_contiguous()):
        raise ValueError("residual must be contiguous, of the result's shape and dtype.")
    if norm_weight is not None:
        if norm_weight.shape != (k,) or norm_weight.device != device or not norm_weight.is_floating_point():
            raise ValueError("norm_weight must be floating-point [k].")
        norm_weight = norm_weight.float().contiguous()  # no copy for the usual float32 vector
        if norm_weight.data_ptr() % 16:
            norm_weight = norm_weight.clone()  # a slice of a larger buffer
    out = x.new_empty(shape)
    rows, lib = x.numel() // k, _capi.lib()
    ws_bytes = 0 if norm_weight is None else lib.hx_int4_workspace_bytes(rows, k, 1)
    workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes else None
    code = _launch(
        device, lib.hx_int4_gemm, x.data_ptr(), k, rows, weight.packed.data_ptr(), weight.steps.data_ptr(), cols, k,
        weight.group, dtype, None if norm_weight is None else norm_weight.data_ptr(), eps,
        None if residual is None else residual.data_ptr(), cols, 1 if swiglu else 0, out.data_ptr(), cols,
        None if workspace is None else workspace.data_ptr(), ws_bytes)
    _capi.check(code, "hx_int4_gemm")
    return out


def int4_dequantize(weight: Int4Weight) -> torch.Tensor:
    """``[rows, k]`` in the weight's dtype: ``scale * (q - zero)``, rounded once."""
    device = _require_gpu(weight.packed)
    dtype = _check_int4(weight, device)
    # Rows of a multiple of 8 elements (k is one of 32), so every row is 16-byte aligned.
    out = torch.empty((weight.rows, weight.k), dtype=weight.dtype, device=device)
    code = _launch(device, _capi.lib().hx_int4_dequantize, weight.packed.data_ptr(), weight.steps.data_ptr(),
                   weight.rows, weight.k, weight.group, dtype, out.data_ptr(), weight.k)
    _capi.check(code, "hx_int4_dequantize")
    return out


# --------------------------------------------------------------------- 8-bit KV cache
_CODES = {torch.float8_e4m3fn: _capi.HX_CODE_E4M3, torch.int8: _capi.HX_CODE_INT8}


class Kv8Cache(NamedTuple):
    """One layer of a paged cache in 8 bits: ``keys`` and ``values`` ``[pages, page_size,
    kv_heads, head_dim]`` float8_e4m3fn or int8, ``key_scales`` and ``value_scales`` float32
    ``[pages, kv_heads, page_size]``, all contiguous. An element stands for its code times the
    scale of its token and head; ``kv8_append`` and ``kv8_norm_rope_append`` write them.
    head_dim is a multiple of 16 up to 256."""

    keys: torch.Tensor
    values: torch.Tensor
    key_scales: torch.Tensor
    value_scales: torch.Tensor


def _check_codes(codes: torch.Tensor, scales: torch.Tensor) -> tuple[int, int, int, int, int]:
    """A code of codes and scales checked: its type's code, pages, page size, KV heads, head dim."""
    code, shape = _CODES.get(codes.dtype), codes.shape
    if code is None:
        raise ValueError("8-bit codes must be float8_e4m3fn or int8.")
    if len(shape) != 4 or 0 in shape or not codes.is_contiguous():
        raise ValueError("8-bit codes must be a contiguous [pages, page_size, kv_heads, head_dim] pool.")
    pages, page_size, n_kv, head_dim = shape
    if head_dim % 16 or head_dim > 256:
        raise ValueError("head_dim of an 8-bit cache must be a multiple of 16 from 16 to 256.")
    if scales.dtype != torch.float32 or scales.shape != (pages, n_kv, page_size) or not scales.is_contiguous():
        raise ValueError("scales must be contiguous float32 [pages, kv_heads, page_size].")
    return code, pages, page_size, n_kv, head_dim


def _check_kv8(cache: Kv8Cache) -> tuple[int, int, int, int, int]:
    keys, values, key_scales, value_scales = cache
    layout = _check_codes(keys, key_scales)
    if values.dtype != keys.dtype or values.shape != keys.shape or not values.is_contiguous() \
            or value_scales.dtype != torch.float32 or value_scales.shape != key_scales.shape \
            or not value_scales.is_contiguous():
        raise ValueError("keys and values of an 8-bit cache must have the same dtypes, shapes and layout.")
    return layout


def _gpu_of(tensors: Sequence[torch.Tensor]) -> torch.device:
    """``_require_gpu`` by the devices' indexes alone: a third of its time for a dozen tensors."""
    index = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != index:
            return _require_gpu(*tensors)
    return tensors[0].device if index >= 0 else _require_gpu(*tensors)


def _check_kv8_rows(keys: torch.Tensor, values: torch.Tensor, write_slots: torch.Tensor, n_kv: int,
                    head_dim: int) -> int:
    """Checks of new keys and values for an 8-bit cache; their dtype code."""
    dtype = _SUPPORTED.get(keys.dtype)
    if dtype is None or values.dtype != keys.dtype:
        raise ValueError("Appended K/V must be bfloat16 or float16, of one dtype.")
    if keys.ndim != 3 or values.shape != keys.shape:
        raise ValueError("Appended keys and values must be [tokens, kv_heads, head_dim].")
    if tuple(keys.shape[1:]) != (n_kv, head_dim):
        raise ValueError("Appended K/V heads do not match the pool layout.")
    if write_slots.dtype != torch.int64 or write_slots.shape != (keys.shape[0],):
        raise ValueError("write_slots must be int64 [tokens].")
    if keys.stride(2) != 1 or values.stride(2) != 1:
        raise ValueError("Appended K/V must have a contiguous head_dim.")
    return dtype


def kv8_append(cache: Kv8Cache, write_slots: torch.Tensor, keys: torch.Tensor, values: torch.Tensor) -> None:
    """``kv_append`` into an 8-bit cache: token t's rows, each with the scale ``max(max |x| * (1 / Q),
    2^-100)`` (Q: 448 for float8_e4m3fn, 127 for int8) and the codes ``x / scale`` rounded to
    nearest even, in fp32 with 1 / Q rounded to it, at slot ``write_slots[t]`` (``page * page_size + offset``; outside the pool:
    skipped; listed twice: one of its tokens, or parts of several). ``keys`` / ``values``
    ``[T, kv_heads, head_dim]`` bfloat16 or float16, any row and head strides. A row with an
    infinite or NaN element is stored as NaN: under a NaN scale."""
    device = _gpu_of((*cache, write_slots, keys, values))
    code, pages, page_size, n_kv, head_dim = _check_kv8(cache)
    dtype = _check_kv8_rows(keys, values, write_slots, n_kv, head_dim)
    write_slots = write_slots.contiguous()
    status = _launch(
        device, _capi.lib().hx_kv8_append, cache.keys.data_ptr(), cache.values.data_ptr(),
        cache.key_scales.data_ptr(), cache.value_scales.data_ptr(), pages, page_size, n_kv, head_dim, code,
        keys.data_ptr(), keys.stride(0), keys.stride(1), values.data_ptr(), values.stride(0), values.stride(1),
        write_slots.data_ptr(), keys.shape[0], dtype)
    _capi.check(status, "hx_kv8_append")


def kv8_norm_rope_append(
    queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, q_norm_weight: torch.Tensor,
    k_norm_weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, cache: Kv8Cache,
    write_slots: torch.Tensor, eps: float, out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``qk_norm_rope_append`` into an 8-bit cache, at any head_dim it holds: RMSNorm and position
    rotation of queries and keys, and the quantised append, in one launch. Returns the
    normalised, rotated queries (``out`` if given), in fp32 and rounded once
    (``qk_norm_rope_append`` rounds between the norm and the rotation, as its reference does).
    Keys, but for the root of their squares' mean, are in fp64 until their scales and codes are
    rounded. Arguments as there, ``write_slots`` as for ``kv8_append``."""
    device = _gpu_of((queries, keys, values, q_norm_weight, k_norm_weight, cos, sin, positions, *cache, write_slots))
    code, pages, page_size, n_kv, head_dim = _check_kv8(cache)
    dtype = _check_kv8_rows(keys, values, write_slots, n_kv, head_dim)
    if queries.ndim != 3 or queries.shape[0] != keys.shape[0] or queries.shape[2] != head_dim or queries.shape[1] < 1:
        raise ValueError("queries must be [tokens, q_heads, head_dim] matching the keys.")
    if queries.dtype != keys.dtype or queries.stride(2) != 1:
        raise ValueError("queries must share the K/V dtype and have a contiguous head_dim.")
    _check_rope(q_norm_weight, k_norm_weight, cos, sin, head_dim)
    if cos.shape[0] < 1:
        raise ValueError("cos/sin need at least one row.")
    tokens, n_q, _ = queries.shape
    if positions.dtype != torch.int64 or positions.numel() != tokens:
        raise ValueError("positions must be int64 with one entry per row.")
    if positions.ndim != 1:
        positions = positions.reshape(-1)
    positions, write_slots = positions.contiguous(), write_slots.contiguous()
    if out is None:
        out = torch.empty((tokens, n_q, head_dim), dtype=queries.dtype, device=device)
    elif out.shape != queries.shape or out.dtype != queries.dtype or out.device != device or out.stride(2) != 1:
        raise ValueError("out must match the queries' shape, dtype and device.")
    tables = [q_norm_weight, k_norm_weight, cos, sin]
    at = [t.data_ptr() for t in tables]
    for i in range(4):
        if at[i] % 16:
            tables[i] = tables[i].clone()
            at[i] = tables[i].data_ptr()
    q_row, q_head, _ = queries.stride()
    k_row, k_head, _ = keys.stride()
    v_row, v_head, _ = values.stride()
    out_row, out_head, _ = out.stride()
    status = _launch(
        device, _capi.lib().hx_kv8_norm_rope_append, queries.data_ptr(), q_row, q_head, keys.data_ptr(), k_row, k_head,
        values.data_ptr(), v_row, v_head, *at, cos.shape[0], positions.data_ptr(), tokens, n_q, n_kv, head_dim, eps, dtype,
        out.data_ptr(), out_row, out_head, cache.keys.data_ptr(), cache.values.data_ptr(),
        cache.key_scales.data_ptr(), cache.value_scales.data_ptr(), pages, page_size, code, write_slots.data_ptr())
    _capi.check(status, "hx_kv8_norm_rope_append")
    return out


def kv8_gather(codes: torch.Tensor, scales: torch.Tensor, pages: torch.Tensor | Sequence[int], length: int,
               dtype: torch.dtype) -> torch.Tensor:
    """``kv_gather`` of an 8-bit pool's keys or values: paged -> dense ``[1, Hkv, length, d]`` in
    ``dtype`` (bfloat16, float16 or float32), ``code * scale`` rounded once."""
    device = _require_gpu(codes, scales)
    code, num_pages, page_size, n_kv, head_dim = _check_codes(codes, scales)
    out_type = _capi.HX_DTYPE_FP32 if dtype == torch.float32 else _SUPPORTED.get(dtype)
    if out_type is None:
        raise ValueError("kv8_gather gives bfloat16, float16 or float32.")
    if not isinstance(pages, torch.Tensor):
        pages = torch.tensor(list(pages), dtype=torch.int32, device=device)
    if pages.ndim != 1 or pages.dtype != torch.int32 or pages.device != device:
        raise ValueError("pages must be an int32 vector on the cache's device.")
    pages = pages.contiguous()
    if length < 0 or length > pages.shape[0] * page_size:
        raise ValueError("length exceeds the listed pages.")
    out = torch.empty((1, n_kv, length, head_dim), dtype=dtype, device=device)
    status = _launch(device, _capi.lib().hx_kv8_gather, codes.data_ptr(), scales.data_ptr(), num_pages, page_size,
                     n_kv, head_dim, code, pages.data_ptr(), pages.shape[0], length, out_type, out.data_ptr())
    _capi.check(status, "hx_kv8_gather")
    return out


class Kv8AttnPlan:
    """``VarlenAttnPlan`` for an 8-bit cache: the work lists of one set of varlen metadata, built
    once per tick, then ``run`` per layer. Query heads that share a KV head: at most 128;
    page_size a multiple of 64. ``q_lens`` (the sequences' new tokens, a host list), when given,
    leaves out launches for kinds of rows that the tick does not have. Runs of one plan share its
    workspace: on several streams, or captured into graphs that may run at once, they need an
    order."""

    def __init__(self, cu_seq_q: torch.Tensor, seqused_k: torch.Tensor, *, total_q: int, max_q: int, max_k: int,
                 n_q_heads: int, n_kv_heads: int, head_dim: int, page_size: int, window: tuple[int, int] = (-1, 0),
                 q_lens: Sequence[int] | None = None, block_table_width: int | None = None) -> None:
        device = _require_gpu(cu_seq_q, seqused_k)
        batch = seqused_k.shape[0] if seqused_k.ndim == 1 else -1
        for name, t, count in (("cu_seq_q", cu_seq_q, batch + 1), ("seqused_k", seqused_k, batch)):
            if t.dtype != torch.int32 or t.shape != (count,):
                raise ValueError(f"{name} must be an int32 vector: batch + 1 and batch entries.")
        if total_q < 0 or max_q < 0 or max_k < 0:
            raise ValueError("total_q, max_q and max_k must be non-negative.")
        if n_kv_heads < 1 or n_q_heads < 1 or n_q_heads % n_kv_heads:
            raise ValueError(f"GQA needs n_q_heads ({n_q_heads}) to be a multiple of n_kv_heads ({n_kv_heads}).")
        if page_size < 1:
            raise ValueError("page_size must be positive.")
        left, right = (max(-1, min(int(x), 2 ** 31 - 1)) for x in window)
        # Without a width the table of every run must cover max_k.
        width = max(1, -(-max_k // page_size)) if block_table_width is None else block_table_width
        lib = _capi.lib()
        self.ws_bytes = lib.hx_kv8_attn_workspace_bytes(batch, total_q, max_q, max_k, n_q_heads, n_kv_heads, head_dim,
                                                        page_size)
        if not self.ws_bytes:
            raise ValueError("Unsupported attention shape: head_dim must be a multiple of 16 from 16 to 256, page_size "
                             "of 64, at most 128 query heads may share a KV head, and batch * max_k stays below 2^36.")
        self.device, self.width = device, width
        self._shape = (batch, total_q, max_q, max_k, n_q_heads, n_kv_heads, head_dim)
        self.page_size, self.window = page_size, (left, right)
        group = n_q_heads // n_kv_heads
        few = max(1, 16 // group)  # rows of a sequence that share one pass over its keys
        self._kinds = _capi.HX_KV8_FEW_ROWS | _capi.HX_KV8_CHUNK_ROWS
        if q_lens is not None:
            kinds = {_capi.HX_KV8_CHUNK_ROWS if n > few else _capi.HX_KV8_FEW_ROWS for n in q_lens if n > 0}
            self._kinds = sum(kinds)
        self._scale = 1.0 / math.sqrt(head_dim)
        self._q_shape = torch.Size((total_q, n_q_heads, head_dim))
        self.workspace = torch.empty(self.ws_bytes + 256, dtype=torch.uint8, device=device)
        self._offset = -self.workspace.data_ptr() % 256
        self._ws_ptr = self.workspace.data_ptr() + self._offset
        cu_seq_q, seqused_k = cu_seq_q.contiguous(), seqused_k.contiguous()
        status = _launch(device, lib.hx_kv8_attn_plan, cu_seq_q.data_ptr(), seqused_k.data_ptr(), *self._shape,
                         page_size, width, left, right, self._ws_ptr, self.ws_bytes)
        _capi.check(status, "hx_kv8_attn_plan")

    def error_word(self) -> int:
        """HX_WERR_* bits raised so far (synchronises the device to read them)."""
        if 0 in self._shape[:3]:
            return 0  # nothing to plan, nothing written
        at = self._offset + _capi.lib().hx_kv8_attn_error_word_offset()
        return int(self.workspace[at:at + 4].view(torch.int32).item())

    def check_errors(self) -> None:
        """Raise RuntimeError if the plan or a run flagged bad metadata (synchronises)."""
        word = self.error_word()
        if word:
            raise RuntimeError(f"8-bit paged attention metadata error {word:#x}: {describe_error_word(word)}")

    def run(self, query: torch.Tensor, cache: Kv8Cache, block_table: torch.Tensor, *, scale: float | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention for one layer: ``query`` ``[total_q, Hq, d]`` bfloat16 or float16, packed, over
        the pages of ``cache`` that ``block_table`` (int32 ``[batch, width]``) lists. Returns
        ``[total_q, Hq, d]`` like ``query``: weights of 22 bits, sums in fp32, rounded once. A row without a
        key gets zeros; output rows behind the last sequence stay as they were. A key or value that was
        stored as NaN makes the rows that see it NaN. A key counts while its weight times its value's
        scale is at least 2^-126 of the row's largest; outputs below 2^-80 may be 0."""
        keys, values, key_scales, value_scales = cache
        device, index = self.device, self.device.index
        for t in (query, keys, values, key_scales, value_scales, block_table):
            if t.get_device() != index:
                _require_gpu(query, *cache, block_table)
                raise ValueError("Query and cache must be on the plan's device.")
        code, pages, page_size, n_kv, head_dim = _check_kv8(cache)
        dtype = _SUPPORTED.get(query.dtype)
        if dtype is None or query.shape != self._q_shape:
            raise ValueError("query must be bfloat16 or float16 [total_q, n_q_heads, head_dim] as planned.")
        if page_size != self.page_size or n_kv != self._shape[5] or head_dim != self._shape[6]:
            raise ValueError("the cache's page size, heads and head_dim must be the planned ones.")
        batch, width, table_stride = _table_layout(block_table)
        if batch != self._shape[0] or width < self.width:
            raise ValueError(f"block_table must be int32 [{self._shape[0]}, {self.width}] or wider, as planned.")
        scale = self._scale if scale is None else float(scale)
        if not 0.0 < scale < math.inf:
            raise ValueError("scale must be positive.")
        if out is None:
            out = torch.empty(self._q_shape, dtype=query.dtype, device=device)
        elif out.shape != query.shape or out.dtype != query.dtype or out.get_device() != index or out.stride(2) != 1 \
                or out.data_ptr() % 4 or out.stride(0) % 2 or out.stride(1) % 2:
            raise ValueError("out must have the query's shape, dtype and device, a contiguous head_dim and even strides.")
        query = _vector_rows(query)
        q_row, q_head, _ = query.stride()
        out_row, out_head, _ = out.stride()
        status = _launch(
            device, _capi.lib().hx_kv8_attn_run, query.data_ptr(), q_row, q_head, keys.data_ptr(), values.data_ptr(),
            key_scales.data_ptr(), value_scales.data_ptr(), pages, page_size, code, block_table.data_ptr(),
            table_stride, self.width, *self._shape, scale, *self.window, dtype, out.data_ptr(), out_row, out_head,
            self._kinds, self._ws_ptr, self.ws_bytes)
        _capi.check(status, "hx_kv8_attn_run")
        if CHECK_ERRORS:
            self.check_errors()
        return out


def kv8_attn(query: torch.Tensor, cache: Kv8Cache, cu_seq_q: torch.Tensor, seqused_k: torch.Tensor,
             block_table: torch.Tensor, *, max_q: int, max_k: int, is_causal: bool = False,
             window_size: tuple[int, int] | None = None, scale: float | None = None) -> torch.Tensor:
    """``varlen_attn`` over an 8-bit paged cache, plan and run in one call. ``window_size=(-1, 0)``
    is the bottom-right causal mask, None every key."""
    device = _require_gpu(query, *cache, cu_seq_q, seqused_k, block_table)
    del device
    _, _, page_size, n_kv, head_dim = _check_kv8(cache)
    if query.ndim != 3:
        raise ValueError("query must be [total_q, n_q_heads, head_dim].")
    _, width, _ = _table_layout(block_table)
    plan = Kv8AttnPlan(cu_seq_q, seqused_k, total_q=query.shape[0], max_q=max_q, max_k=max_k,
                       n_q_heads=query.shape[1], n_kv_heads=n_kv, head_dim=head_dim, page_size=page_size,
                       window=_window(window_size, is_causal), block_table_width=width)
    return plan.run(query, cache, block_table, scale=scale)


# --------------------------------------------------------------- rules on the logits
class LogitRules(NamedTuple):
    """What the requests of a tick ask of their logit rows, all on the device, None: not asked.

    ``tokens`` int32 ``[rows, cap]`` with ``lengths`` int32 ``[rows]``: the tokens row r knows
    are ``tokens[r, :lengths[r]]`` (a server appends a column a tick), the first
    ``prompt_lens[r]`` (int32, None: 0) its prompt, the others said. ``repetition`` (of
    known tokens), ``presence`` and ``frequency`` (of said ones): float32 ``[rows]``.
    ``bias_ids`` int32 and ``bias_values`` float32 ``[rows, n]``, of one row stride: added to
    those tokens; of an id listed twice in a row the last counts. ``allowed`` int32 ``[rows, ceil(vocab / 32)]``:
    bit ``v % 32`` of word ``v // 32`` allows token v. Token and bias ids outside the
    vocabulary (-1: padding) are skipped. Rows of a table are contiguous and do not overlap."""

    tokens: torch.Tensor | None = None
    lengths: torch.Tensor | None = None
    prompt_lens: torch.Tensor | None = None
    repetition: torch.Tensor | None = None
    presence: torch.Tensor | None = None
    frequency: torch.Tensor | None = None
    bias_ids: torch.Tensor | None = None
    bias_values: torch.Tensor | None = None
    allowed: torch.Tensor | None = None


class RuledLogits(NamedTuple):
    """Result of ``apply_logit_rules``: ``logits`` in the input's shape and dtype (None when
    not asked for) and the greedy ``token_ids`` int64 ``[rows]``."""

    logits: torch.Tensor | None
    token_ids: torch.Tensor


_RULE_KINDS = ((torch.int32, 2), (torch.int32, 1), (torch.int32, 1), (torch.float32, 1), (torch.float32, 1),
               (torch.float32, 1), (torch.int32, 2), (torch.float32, 2), (torch.int32, 2))  # of LogitRules' fields


def _check_rules(rules: LogitRules, rows: int, vocab: int, device: torch.device) -> None:
    for i, (t, (dtype, ndim)) in enumerate(zip(rules, _RULE_KINDS)):
        if t is None:
            continue
        shape = t.shape
        if ndim == 1:
            if t.dtype != dtype or shape != (rows,) or not t.is_contiguous():
                raise ValueError(f"{rules._fields[i]} must be contiguous {dtype} [{rows}].")
        elif t.dtype != dtype or len(shape) != 2 or shape[0] != rows or not t.is_contiguous() and (
                (shape[1] > 1 and t.stride(1) != 1) or (rows > 1 and t.stride(0) < shape[1])):
            raise ValueError(f"{rules._fields[i]} must be {dtype} [{rows}, n] with contiguous rows.")
        if t.device != device:
            raise ValueError(f"{rules._fields[i]} must be on the logits' device.")
    tokens, lengths, prompt_lens, repetition, presence, frequency, bias_ids, bias_values, allowed = rules
    if (tokens is None) != (lengths is None):
        raise ValueError("tokens and lengths go together.")
    if tokens is None and any(t is not None for t in (prompt_lens, repetition, presence, frequency)):
        raise ValueError("prompt_lens, repetition, presence and frequency need tokens.")
    if (bias_ids is None) != (bias_values is None) or (bias_ids is not None and bias_ids.shape != bias_values.shape):
        raise ValueError("bias_ids and bias_values go together, in one shape.")
    if bias_ids is not None and rows > 1 and bias_ids.stride(0) != bias_values.stride(0):
        raise ValueError("bias_ids and bias_values must have the same row stride.")
    if allowed is not None and allowed.shape[1] < -(-vocab // 32):
        raise ValueError("allowed needs a bit for every token of the vocabulary.")


def apply_logit_rules(logits: torch.Tensor, rules: LogitRules, *, out: torch.Tensor | None = None,
                      return_logits: bool = True) -> RuledLogits:
    """Penalties, biases and allowed tokens on ``logits`` ``[rows, vocab]`` (bfloat16, float16
    or float32, contiguous rows), and the greedy ids of the result.

    In fp32, each step rounded, for a token v of row r with logit l: known,
    ``l / repetition`` if l > 0, else ``l * repetition``; said c times,
    ``l - (frequency * c + presence)``; listed, ``l + bias``; not allowed, ``-inf``; then
    rounded to the dtype. ``token_ids[r]`` is the smallest allowed token with the largest
    result (a NaN counts as the largest, as in ``torch.argmax``), -1 in a row that nothing
    is allowed in. ``out`` may be ``logits`` itself (in place), or memory that does not
    overlap it; with ``return_logits=False`` and no ``out`` only the ids are written."""
    device = _require_gpu(logits)
    dtype = _capi.HX_DTYPE_FP32 if logits.dtype == torch.float32 else _SUPPORTED.get(logits.dtype)
    if dtype is None or logits.ndim != 2 or logits.shape[1] < 1:
        raise ValueError("logits must be bfloat16, float16 or float32 [rows, vocab].")
    rows, vocab = logits.shape
    if (vocab > 1 and logits.stride(1) != 1) or (rows > 1 and logits.stride(0) < vocab):
        raise ValueError("logits need contiguous rows that do not overlap.")
    _check_rules(rules, rows, vocab, device)
    if out is None:
        if return_logits:
            out = logits.new_empty((rows, vocab))
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != device \
            or (vocab > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < vocab):
        raise ValueError("out must have the logits' shape, dtype and device, and contiguous rows.")
    elif out.data_ptr() == logits.data_ptr() and rows > 1 and out.stride(0) != logits.stride(0):
        raise ValueError("out must be the logits or memory that does not overlap them.")
    token_ids = logits.new_empty(rows, dtype=torch.int64)
    if rows == 0:
        return RuledLogits(out, token_ids)
    lib = _capi.lib()
    ws_bytes = lib.hx_logit_rules_workspace_bytes(rows, vocab)
    workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=device)

    tokens, lengths, prompt_lens, repetition, presence, frequency, bias, bias_values, allowed = [
        None if t is None else t.data_ptr() for t in rules]
    cap = n_bias = words = token_stride = bias_stride = 0
    if tokens is not None:
        cap = rules.tokens.shape[1]
        token_stride = rules.tokens.stride(0) if rows > 1 else cap  # a single row's stride may be anything
    if bias is not None:
        n_bias = rules.bias_ids.shape[1]
        bias_stride = rules.bias_ids.stride(0) if rows > 1 else n_bias
    if allowed is not None:
        words = rules.allowed.stride(0) if rows > 1 else rules.allowed.shape[1]
    code = _launch(
        device, lib.hx_logit_rules, logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, rows, vocab, dtype,
        tokens if cap else None, token_stride, cap, lengths, prompt_lens, repetition, presence, frequency,
        bias if n_bias else None, bias_values, bias_stride, n_bias, allowed, words,
        None if out is None else out.data_ptr(), vocab if out is None or rows == 1 else out.stride(0),
        token_ids.data_ptr(), workspace.data_ptr(), ws_bytes)
    _capi.check(code, "hx_logit_rules")
    return RuledLogits(out, token_ids)


# ------------------------------------------------------------------- drawing tokens
SAMPLE_MAX_VOCAB = 1 << 18  # tokens that sample_tokens can draw from


class SampledTokens(NamedTuple):
    """Result of ``sample_tokens``: ``token_ids`` int64 ``[rows]`` and ``logprobs`` float32
    ``[rows]``, the logarithm of the token's share of the weights that were kept."""

    token_ids: torch.Tensor
    logprobs: torch.Tensor


class Sampling(NamedTuple):
    """How the requests of a tick draw their tokens, a value per logit row: ``sample_tokens``'s
    arguments, for callers that pass them on."""

    uniforms: torch.Tensor
    temperature: torch.Tensor | None = None
    top_k: torch.Tensor | None = None
    top_p: torch.Tensor | None = None
    min_p: torch.Tensor | None = None


def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, *, temperature: torch.Tensor | None = None,
                  top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None,
                  min_p: torch.Tensor | None = None) -> SampledTokens:
    """A token drawn from each row of ``logits`` ``[rows, vocab]`` (bfloat16, float16 or float32,
    contiguous rows) by the numbers ``uniforms`` (float32 ``[rows]``, in [0, 1)).

    With t = ``temperature[r]`` a token's weight is ``exp((logit - largest) / t)``. In order of
    falling logit (equal ones: the lower id first) the first n tokens are kept: at most
    ``top_k[r]`` (int32; 0 or less: all), no more than it takes to reach ``top_p[r]`` of the
    weight of the first ``top_k``, those with a weight of at least ``min_p[r]``, and at least
    one. The token drawn is the first in that order whose cumulative weight passes ``uniforms[r]``
    of theirs. A temperature of 0 or less takes the first token (as ``torch.argmax``, logprob 0), as
    does a row whose largest logit is +inf or NaN; a row of -inf alone gives -1 and -inf. Limits are
    float32 (``top_k`` int32) ``[rows]``, None: none; a ``temperature`` of None is 1, and others are held
    to [1e-30, 1e30]. Weights are within 2^-44.6 of the largest, those below 2^-45 of it count as 0, and
    sums of them have no order: equal inputs give equal tokens."""
    device = _require_gpu(logits, uniforms)
    dtype = _capi.HX_DTYPE_FP32 if logits.dtype == torch.float32 else _SUPPORTED.get(logits.dtype)
    if dtype is None or logits.ndim != 2 or logits.shape[1] < 1:
        raise ValueError("logits must be bfloat16, float16 or float32 [rows, vocab].")
    rows, vocab = logits.shape
    if vocab > SAMPLE_MAX_VOCAB:
        raise ValueError(f"sample_tokens draws from at most {SAMPLE_MAX_VOCAB} tokens.")
    if (vocab > 1 and logits.stride(1) != 1) or (rows > 1 and logits.stride(0) < vocab):
        raise ValueError("logits need contiguous rows that do not overlap.")
    index = device.index
    for name, t, kind in (("uniforms", uniforms, torch.float32), ("temperature", temperature, torch.float32),
                          ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32),
                          ("min_p", min_p, torch.float32)):
        if t is not None and (t.dtype != kind or t.shape != (rows,) or not t.is_contiguous() or t.get_device() != index):
            raise ValueError(f"{name} must be contiguous {kind} [{rows}] on the logits' device.")
    token_ids = logits.new_empty(rows, dtype=torch.int64)
    logprobs = logits.new_empty(rows, dtype=torch.float32)
    if rows == 0:
        return SampledTokens(token_ids, logprobs)
    lib = _capi.lib()
    ws_bytes = lib.hx_sample_workspace_bytes(rows, vocab)
    workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
    code = _launch(
        device, lib.hx_sample_tokens, logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, rows, vocab, dtype,
        uniforms.data_ptr(), *(None if t is None else t.data_ptr() for t in (temperature, top_k, top_p, min_p)),
        token_ids.data_ptr(), logprobs.data_ptr(), workspace.data_ptr(), ws_bytes)
    _capi.check(code, "hx_sample_tokens")
    return SampledTokens(token_ids, logprobs)


# --------------------------------------------------------------- logits and argmax
class GreedyHeads(NamedTuple):
    """Result of ``final_norm_logits_argmax``: ``token_ids`` int64 ``[n]`` (-1 for an index
    outside the hidden rows), ``max_logits`` fp32 ``[n]``, and ``logits`` ``[n, vocab]``
    in the model dtype when they were asked for (else None)."""

    token_ids: torch.Tensor
    max_logits: torch.Tensor
    logits: torch.Tensor | None


def final_norm_logits_argmax(
    hidden_states: torch.Tensor,
    logit_indices: torch.Tensor,
    norm_weight: torch.Tensor,
    embedding: torch.Tensor,
    eps: float,
    *,
    return_logits: bool = False,
) -> GreedyHeads:
    """Greedy heads of a packed tick: the final RMSNorm of the logit rows, the tied
    lm_head and argmax, replacing ``x.index_select(1, logit_indices)``,
    ``self.output(self.final_norm(x).to(dtype))`` (model.py:108-110) and
    ``heads.argmax(dim=-1)`` (engine.py:470-473) for greedy sampling.

    ``hidden_states`` ``[T, hidden]`` or ``[1, T, hidden]`` (the last layer's output,
    contiguous last dim); ``logit_indices`` int64 ``[n]``; ``norm_weight`` fp32
    ``[hidden]``; ``embedding`` ``[vocab, hidden]`` in the model dtype. Ties go to the
    smallest vocab index, as in ``torch.argmax``. The logits are computed in fp32,
    rounded to the model dtype like the Linear's output, and written out only with
    ``return_logits``.
    """
    if hidden_states.ndim == 3:
        if hidden_states.shape[0] != 1:
            raise ValueError("hidden_states must be [tokens, hidden] or [1, tokens, hidden].")
        hidden_states = hidden_states[0]
    device = _require_gpu(hidden_states, logit_indices, norm_weight, embedding)
    if hidden_states.ndim != 2 or embedding.ndim != 2 or embedding.shape[1] != hidden_states.shape[1]:
        raise ValueError("embedding must be [vocab, hidden] matching hidden_states.")
    if hidden_states.dtype != embedding.dtype:
        raise ValueError("hidden_states and embedding must share a dtype.")
    dtype = _SUPPORTED.get(embedding.dtype)
    if dtype is None:
        raise ValueError("hidden_states and embedding must be bfloat16 or float16.")
    if hidden_states.stride(1) != 1 or embedding.stride(1) != 1:
        raise ValueError("hidden_states and embedding need a contiguous last dimension.")
    hidden = hidden_states.shape[1]
    if norm_weight.dtype != torch.float32 or tuple(norm_weight.shape) != (hidden,) or not norm_weight.is_contiguous():
        raise ValueError("norm_weight must be contiguous float32 [hidden].")
    if logit_indices.dtype != torch.int64 or logit_indices.ndim != 1 or not logit_indices.is_contiguous():
        raise ValueError("logit_indices must be contiguous int64 [n].")
    n, vocab = logit_indices.numel(), embedding.shape[0]
    token_ids = torch.empty(n, dtype=torch.int64, device=device)
    max_logits = torch.empty(n, dtype=torch.float32, device=device)
    logits = torch.empty((n, vocab), dtype=embedding.dtype, device=device) if return_logits else None
    if n == 0:
        return GreedyHeads(token_ids, max_logits, logits)
    lib = _capi.lib()
    ws_bytes = lib.hx_logits_workspace_bytes(n, vocab, hidden)
    workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
    code = lib.hx_final_norm_logits_argmax(
        hidden_states.data_ptr(), hidden_states.stride(0), hidden_states.shape[0],
        logit_indices.data_ptr(), n, norm_weight.data_ptr(), float(eps),
        embedding.data_ptr(), embedding.stride(0), vocab, hidden, dtype,
        token_ids.data_ptr(), max_logits.data_ptr(),
        logits.data_ptr() if logits is not None else None, vocab,
        workspace.data_ptr(), ws_bytes, _stream_ptr(device),
    )
    _capi.check(code, "hx_final_norm_logits_argmax")
    return GreedyHeads(token_ids, max_logits, logits)


# --------------------------------------------------------------- tick metadata
def tick_metadata(
    seq: torch.Tensor,
    block_table: torch.Tensor,
    page_size: int,
    *,
    total_q: int,
    cu_seq_q: torch.Tensor,
    cu_seq_k: torch.Tensor,
    seqused_k: torch.Tensor,
    write_slots: torch.Tensor,
    positions: torch.Tensor | None = None,
    logit_indices: torch.Tensor | None = None,
    n_logits: int = 0,
) -> None:
    """Per-tick metadata of ``PagedBatchCache.prepare`` / ``PackedBatchCache.prepare_packed``
    (paged_cache.py:221-270, :418-494) computed on the device.

    ``seq``: int32 ``[3 * B]`` = lengths before the tick, tokens this tick, logit rows.
    Writes ``cu_seq_q`` / ``cu_seq_k`` (int32 ``[B+1]``), ``seqused_k`` (int32 ``[B]``),
    ``write_slots`` and optionally ``positions`` (int64, ``total_q`` rows) and
    ``logit_indices`` (int64, ``n_logits`` rows), all preallocated on the device.
    """
    device = _require_gpu(seq, block_table, cu_seq_q, cu_seq_k, seqused_k, write_slots)
    batch = seq.numel() // 3
    if seq.dtype != torch.int32 or seq.numel() != 3 * batch or batch < 1 or not seq.is_contiguous():
        raise ValueError("seq must be a contiguous int32 tensor of 3 * batch values.")
    if block_table.dtype != torch.int32 or block_table.ndim != 2 or block_table.shape[0] != batch:
        raise ValueError("block_table must be int32 [batch, width].")
    if block_table.stride(1) != 1:
        raise ValueError("block_table rows must be contiguous.")
    for name, t, n, dt in (("cu_seq_q", cu_seq_q, batch + 1, torch.int32),
                           ("cu_seq_k", cu_seq_k, batch + 1, torch.int32),
                           ("seqused_k", seqused_k, batch, torch.int32),
                           ("write_slots", write_slots, total_q, torch.int64)):
        if t.dtype != dt or t.numel() < n or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {dt} tensor of at least {n} values.")
    for name, t, n in (("positions", positions, total_q), ("logit_indices", logit_indices, n_logits)):
        if t is not None and (t.dtype != torch.int64 or t.numel() < n or not t.is_contiguous()
                              or t.device != device):
            raise ValueError(f"{name} must be a contiguous int64 tensor of at least {n} values.")
    if n_logits > 0 and logit_indices is None:
        raise ValueError("logit_indices is required when n_logits > 0.")
    code = _capi.lib().hx_tick_metadata(
        seq.data_ptr(), batch, total_q, n_logits,
        block_table.data_ptr(), block_table.stride(0), page_size,
        cu_seq_q.data_ptr(), cu_seq_k.data_ptr(), seqused_k.data_ptr(),
        positions.data_ptr() if positions is not None else None,
        write_slots.data_ptr(),
        logit_indices.data_ptr() if logit_indices is not None else None,
        _stream_ptr(device),
    )
    _capi.check(code, "hx_tick_metadata")


# --------------------------------------------------------------------- page copy
def kv_copy_pages(
    k_caches: Sequence[torch.Tensor],
    v_caches: Sequence[torch.Tensor] | None,
    src_pages: Sequence[int],
    dst_pages: Sequence[int],
) -> None:
    """Copy whole pages for every layer: ``cache[l][dst[i]] = cache[l][src[i]]``.

    Bit-exact; the page-granular form of KVCache.snapshot_block/restore_blocks
    (cache.py:109-147). ``src_pages``/``dst_pages`` are host lists; destinations
    must be distinct and disjoint from the sources.
    """
    if len(src_pages) != len(dst_pages):
        raise ValueError("Source and destination page lists differ in length.")
    if not k_caches:
        return
    tensors = list(k_caches) + (list(v_caches) if v_caches is not None else [])
    device = _require_gpu(*tensors)
    shape, dtype = k_caches[0].shape, k_caches[0].dtype
    if v_caches is not None and len(v_caches) != len(k_caches):
        raise ValueError("Key and value layer lists differ in length.")
    for t in tensors:
        if t.shape != shape or t.dtype != dtype or not t.is_contiguous():
            raise ValueError("Every pool tensor must share one contiguous [pages, ...] layout.")
    n_layers, n_pages = len(k_caches), len(src_pages)
    if n_pages == 0:
        return
    page_bytes = k_caches[0][0].numel() * k_caches[0].element_size()
    k_ptrs = (ctypes.c_void_p * n_layers)(*[t.data_ptr() for t in k_caches])
    v_ptrs = (
        (ctypes.c_void_p * n_layers)(*[t.data_ptr() for t in v_caches])
        if v_caches is not None
        else None
    )
    src = (ctypes.c_int32 * n_pages)(*[int(p) for p in src_pages])
    dst = (ctypes.c_int32 * n_pages)(*[int(p) for p in dst_pages])
    code = _capi.lib().hx_kv_copy_pages(
        k_ptrs, v_ptrs, n_layers, src, dst, n_pages, shape[0], page_bytes, _stream_ptr(device)
    )
    _capi.check(code, "hx_kv_copy_pages")


# --------------------------------------------------------------------- page gather
def kv_gather(cache: torch.Tensor, pages: torch.Tensor | Sequence[int], length: int) -> torch.Tensor:
    """Paged -> dense ``[1, Hkv, length, d]`` (``_gather_cpu``, paged_cache.py:405-414)."""
    device = _require_gpu(cache)
    if cache.ndim != 4 or not cache.is_contiguous():
        raise ValueError("cache must be a contiguous [pages, page_size, kv_heads, head_dim] pool.")
    num_pages, page_size, n_kv, head_dim = cache.shape
    if not isinstance(pages, torch.Tensor):
        pages = torch.tensor(list(pages), dtype=torch.int32, device=device)
    if pages.ndim != 1 or pages.dtype != torch.int32 or pages.device != device:
        raise ValueError("pages must be an int32 vector on the cache's device.")
    pages = pages.contiguous()
    if length < 0 or length > pages.shape[0] * page_size:
        raise ValueError("length exceeds the listed pages.")
    out = torch.empty((1, n_kv, length, head_dim), dtype=cache.dtype, device=device)
    code = _capi.lib().hx_kv_gather(
        cache.data_ptr(), num_pages, page_size, n_kv, head_dim, cache.element_size(),
        pages.data_ptr(), pages.shape[0], length, out.data_ptr(), _stream_ptr(device),
    )
    _capi.check(code, "hx_kv_gather")
    return out


# --------------------------------------------------------------------- attention
def _window(window_size, is_causal: bool) -> tuple[int, int]:
    if window_size is None:
        return (-1, 0) if is_causal else (-1, -1)
    left, right = (int(x) for x in window_size)
    if is_causal:
        right = 0 if right < 0 else min(right, 0)
    return left, right


def workspace_bytes(batch: int, max_q: int, max_k: int, n_q_heads: int, n_kv_heads: int, head_dim: int) -> int:
    nbytes = _capi.lib().hx_varlen_attn_workspace_bytes(batch, max_q, max_k, n_q_heads, n_kv_heads, head_dim)
    if nbytes == 0:
        raise ValueError(
            "Unsupported attention shape: head_dim must be a multiple of 8 from 8 to 256 and "
            "n_q_heads a multiple of n_kv_heads."
        )
    return nbytes


def count_items(q_lens: Sequence[int], k_lens: Sequence[int], n_q_heads: int, n_kv_heads: int,
                window: tuple[int, int]) -> tuple[int, int, int]:
    """Exact work-item counts the device planner will produce for these lengths."""
    batch = len(q_lens)
    ql = (ctypes.c_int32 * max(batch, 1))(*q_lens)
    kl = (ctypes.c_int32 * max(batch, 1))(*k_lens)
    nd, np_, nc = ctypes.c_int32(), ctypes.c_int32(), ctypes.c_int32()
    code = _capi.lib().hx_varlen_attn_count_items(
        ql, kl, batch, n_q_heads, n_kv_heads, window[0], window[1],
        ctypes.byref(nd), ctypes.byref(np_), ctypes.byref(nc),
    )
    _capi.check(code, "hx_varlen_attn_count_items")
    return nd.value, np_.value, nc.value


class VarlenAttnPlan:
    """Work plan for one set of varlen metadata, reusable across layers.

    Built once per tick (the reference's metadata is identical for all 36 layers),
    then ``run`` is called per layer. ``q_lens``/``k_lens`` (host lists), when given,
    size the launch grids exactly; otherwise the bounds from (batch, max_q, max_k)
    are used and surplus workgroups exit at once.
    """

    def __init__(
        self,
        cu_seq_q: torch.Tensor,
        cu_seq_k: torch.Tensor | None,
        seqused_k: torch.Tensor | None,
        *,
        total_q: int,
        max_q: int,
        max_k: int,
        n_q_heads: int,
        n_kv_heads: int,
        head_dim: int,
        page_size: int,
        block_table_stride: int,
        total_k_rows: int = 0,
        window: tuple[int, int] = (-1, 0),
        q_lens: Sequence[int] | None = None,
        k_lens: Sequence[int] | None = None,
    ) -> None:
        device = _require_gpu(cu_seq_q)
        for name, t in (("cu_seq_q", cu_seq_q), ("cu_seq_k", cu_seq_k), ("seqused_k", seqused_k)):
            if t is None:
                continue
            if t.dtype != torch.int32 or t.ndim != 1 or t.device != device:
                raise ValueError(f"{name} must be an int32 vector on the query's device.")
        batch = cu_seq_q.shape[0] - 1
        if batch < 0:
            raise ValueError("cu_seq_q must have batch + 1 entries.")
        if cu_seq_k is not None and cu_seq_k.shape[0] != batch + 1:
            raise ValueError("cu_seq_k must have batch + 1 entries.")
        if seqused_k is not None and seqused_k.shape[0] != batch:
            raise ValueError("seqused_k must have batch entries.")
        if seqused_k is None and cu_seq_k is None:
            raise ValueError("Either seqused_k or cu_seq_k is required.")
        if max_q < 0 or max_k < 0:
            raise ValueError("max_q and max_k must be non-negative.")
        self.device = device
        self.batch = batch
        self.total_q = total_q
        self.max_q = max_q
        self.max_k = max_k
        self.n_q_heads = n_q_heads
        self.n_kv_heads = n_kv_heads
        self.head_dim = head_dim
        self.page_size = page_size
        self.block_table_stride = block_table_stride
        self.window = window
        # The tuned kernels (split-K decode, MFMA chunk, combine) serve head_dim 128 with
        # 1, 2, 4 or 8 query heads per KV head; other shapes run one kernel for every row and
        # one that merges their splits.
        self.tuned = head_dim == 128 and n_kv_heads > 0 and n_q_heads % n_kv_heads == 0 \
            and n_q_heads // n_kv_heads in (1, 2, 4, 8)
        self._metadata = (cu_seq_q.contiguous(), None if cu_seq_k is None else cu_seq_k.contiguous(),
                          None if seqused_k is None else seqused_k.contiguous())
        self.ws_bytes = workspace_bytes(max(batch, 0), max_q, max_k, n_q_heads, n_kv_heads, head_dim)
        try:
            self.workspace = torch.empty(self.ws_bytes + 256, dtype=torch.uint8, device=device)
        except torch.OutOfMemoryError:
            # Without room for fp32 partials the untuned shapes run in less (whole rows).
            least = workspace_bytes(max(batch, 0), max_q, max_k, n_q_heads, n_kv_heads, 8)
            if self.tuned or least >= self.ws_bytes:
                raise
            self.ws_bytes = least
            self.workspace = torch.empty(self.ws_bytes + 256, dtype=torch.uint8, device=device)
        base = self.workspace.data_ptr()
        self._ws_offset = (-base) % 256
        self.ws_ptr = base + self._ws_offset
        if q_lens is not None and k_lens is not None:
            self.hints = count_items(q_lens, k_lens, n_q_heads, n_kv_heads, window)
        else:
            self.hints = (-1, -1, -1)
        # What append_attend compares its tensors with.
        self._scale = 1.0 / math.sqrt(head_dim)
        self._q_shape = torch.Size((1, n_q_heads, total_q, head_dim))
        self._kv_shape = torch.Size((1, n_kv_heads, total_q, head_dim))
        self._page_shape = torch.Size((page_size, n_kv_heads, head_dim))
        self._page_stride = (page_size * n_kv_heads * head_dim, n_kv_heads * head_dim, head_dim, 1)
        self._table_shape = torch.Size((max(batch, 0), block_table_stride))
        self._out_stride = (n_q_heads * head_dim, head_dim, n_q_heads * head_dim, 1)
        cu_q, cu_k, used = self._metadata
        code = _capi.lib().hx_varlen_attn_plan(
            cu_q.data_ptr(),
            None if cu_k is None else cu_k.data_ptr(),
            None if used is None else used.data_ptr(),
            batch, total_q, max_q, max_k, total_k_rows, page_size, block_table_stride,
            n_q_heads, n_kv_heads, head_dim, window[0], window[1],
            self.ws_ptr, self.ws_bytes, _stream_ptr(device),
        )
        _capi.check(code, "hx_varlen_attn_plan")

    def error_word(self) -> int:
        """HX_WERR_* bits raised so far (synchronises the device to read them)."""
        off = self._ws_offset + _capi.lib().hx_varlen_attn_error_word_offset()
        return int(self.workspace[off:off + 4].view(torch.int32).item())

    def check_errors(self) -> None:
        """Raise RuntimeError if the plan or a run flagged bad metadata (synchronises)."""
        word = self.error_word()
        if word:
            raise RuntimeError(f"paged attention metadata error {word:#x}: {describe_error_word(word)}")

    def append_attend(self, queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                      k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                      write_slots: torch.Tensor) -> torch.Tensor | None:
        """``run(append=...)`` of one layer for the layout the decoder's projections have:
        queries ``[1, Hq, total_q, d]``, keys / values ``[1, Hkv, total_q, d]`` (any row and
        head strides), contiguous pools; returns ``[1, Hq, total_q, d]`` (packed rows in
        memory), without making row views on the way. The same launches and bits. None, and
        nothing launched, for any other layout, type or device: the caller then takes ``run``.

        A short tick's call is bound by this host path. 1 request of 300 keys: 26.4 us a
        call through the row views and ``run``."""
        dtype, index = queries.dtype, self.device.index
        code = _SUPPORTED.get(dtype)
        if (code is None or CHECK_ERRORS or self.page_size <= 0
                or queries.shape != self._q_shape or keys.shape != self._kv_shape or values.shape != self._kv_shape
                or keys.dtype is not dtype or values.dtype is not dtype
                or k_cache.dtype is not dtype or v_cache.dtype is not dtype
                or k_cache.ndim != 4 or k_cache.shape[1:] != self._page_shape or v_cache.shape != k_cache.shape
                or k_cache.stride() != self._page_stride or v_cache.stride() != self._page_stride
                or block_table.dtype is not torch.int32 or block_table.shape != self._table_shape
                or block_table.stride() != (self.block_table_stride, 1)
                or write_slots.dtype is not torch.int64 or write_slots.ndim != 1
                or write_slots.numel() != self.total_q or write_slots.stride(0) != 1
                or queries.get_device() != index or keys.get_device() != index or values.get_device() != index
                or k_cache.get_device() != index or v_cache.get_device() != index
                or block_table.get_device() != index or write_slots.get_device() != index):
            return None
        qs, ks, vs = queries.stride(), keys.stride(), values.stride()
        q_ptr, k_ptr, v_ptr = queries.data_ptr(), keys.data_ptr(), values.data_ptr()
        # 16-byte loads of the new rows, and of q (whose run raises otherwise).
        if (qs[3] != 1 or ks[3] != 1 or vs[3] != 1 or (q_ptr | k_ptr | v_ptr) & 15
                or (qs[1] | qs[2] | ks[1] | ks[2] | vs[1] | vs[2]) & 7):
            return None
        pages, page_size, heads, dim = k_cache.shape
        out = torch.empty_strided(self._q_shape, self._out_stride, dtype=dtype, device=self.device)
        status = _capi.lib().hx_varlen_attn_call(_capi.ATTN_CALL.pack(
            _capi.ATTN_CALL.size, q_ptr, qs[2], qs[1], k_cache.data_ptr(), v_cache.data_ptr(), heads * dim, dim,
            pages, page_size, block_table.data_ptr(), self.block_table_stride,
            self.batch, self.total_q, self.max_q, self.max_k, self.n_q_heads, heads, dim,
            self._scale, self.window[0], self.window[1], code, out.data_ptr(), self._out_stride[0], dim, 0,
            k_ptr, ks[2], ks[1], v_ptr, vs[2], vs[1], write_slots.data_ptr(), pages * page_size,
            *self.hints, self.ws_ptr, self.ws_bytes), torch._C._cuda_getCurrentRawStream(index))
        _capi.check(status, "hx_varlen_attn_call")
        return out

    def attend_rows(self, query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_table: torch.Tensor) -> torch.Tensor | None:
        """``run(query, ...)`` without its options, for contiguous packed queries
        ``[total_q, Hq, d]`` and contiguous pools; None, and nothing launched, otherwise."""
        dtype, index = query.dtype, self.device.index
        code = _SUPPORTED.get(dtype)
        if (code is None or CHECK_ERRORS or self.page_size <= 0
                or query.ndim != 3 or query.shape[0] != self.total_q or query.shape[1] != self.n_q_heads
                or query.shape[2] != self.head_dim or not query.is_contiguous()
                or k_cache.dtype is not dtype or v_cache.dtype is not dtype
                or k_cache.ndim != 4 or k_cache.shape[1:] != self._page_shape or v_cache.shape != k_cache.shape
                or k_cache.stride() != self._page_stride or v_cache.stride() != self._page_stride
                or block_table.dtype is not torch.int32 or block_table.shape != self._table_shape
                or block_table.stride() != (self.block_table_stride, 1)
                or query.get_device() != index or k_cache.get_device() != index or v_cache.get_device() != index
                or block_table.get_device() != index):
            return None
        pages, page_size, heads, dim = k_cache.shape
        row = self._out_stride[0]
        out = torch.empty_like(query)
        status = _capi.lib().hx_varlen_attn_call(_capi.ATTN_CALL.pack(
            _capi.ATTN_CALL.size, query.data_ptr(), row, dim, k_cache.data_ptr(), v_cache.data_ptr(), heads * dim, dim,
            pages, page_size, block_table.data_ptr(), self.block_table_stride,
            self.batch, self.total_q, self.max_q, self.max_k, self.n_q_heads, heads, dim,
            self._scale, self.window[0], self.window[1], code, out.data_ptr(), row, dim, 0,
            0, 0, 0, 0, 0, 0, 0, 0, *self.hints, self.ws_ptr, self.ws_bytes),
            torch._C._cuda_getCurrentRawStream(index))
        _capi.check(status, "hx_varlen_attn_call")
        return out

    def run(
        self,
        query: torch.Tensor,
        k_cache: torch.Tensor,
        v_cache: torch.Tensor,
        block_table: torch.Tensor | None,
        *,
        scale: float | None = None,
        out: torch.Tensor | None = None,
        return_lse: bool = False,
        lse_out: torch.Tensor | None = None,
        phases: tuple[str, ...] = ("decode", "chunk", "combine"),
        append: tuple[torch.Tensor, torch.Tensor, torch.Tensor] | None = None,
        query_rows: torch.Tensor | None = None,
        merge: MergeParts | None = None,
    ) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
        """Attention for one layer. ``phases`` launches a subset of the three kernels
        (decode splits, chunk rows, split combine); a full result needs all three, with
        the combine after the other two (the launch order within one call), into the
        same ``out`` (and ``lse_out``, when the log-sum-exp is wanted). Profilers use it
        to time each kernel, and ``run_overlapped`` to run decode and chunk rows on two
        streams.

        ``append=(k_new, v_new, write_slots)`` first writes the tick's new K/V rows
        into the pool (index_copy_ semantics, as ``kv_append``) in the same call: decode
        rows inside the decode kernel, chunk rows by the append kernel beforehand.

        ``query_rows`` (int64 ``[total_q]`` on the device) reads packed row t's query
        from ``query[query_rows[t]]``, so ``query`` may be any ``[N, n_q_heads,
        head_dim]``; ``out`` and the log-sum-exp stay ``[total_q, ...]``. It is the
        result of ``run(query.index_select(0, query_rows), ...)`` without the gather. An
        entry outside ``[0, N)`` reads row 0 and sets an error-word bit. Not combined
        with ``append``.

        ``merge`` (``MergeParts``) folds a shared-prefix cascade's level results into its
        members' rows inside the combine launch: the bits of this run followed by
        ``attn_merge`` over the same parts, one launch fewer. It needs the combine phase
        and the log-sum-exp output (``return_lse`` or ``lse_out``), on the tuned shapes.
        """
        _require_gpu(query, k_cache, v_cache)
        unknown = set(phases) - {"decode", "combine", "chunk"}
        if unknown:
            raise ValueError(f"unknown attention phases {sorted(unknown)}")
        if query.device != self.device:
            raise ValueError("Query is not on the plan's device.")
        if query.dtype not in _SUPPORTED:
            raise ValueError("varlen_attn supports bfloat16 and float16 queries.")
        rows_in = self.total_q if query_rows is None else query.shape[0]
        if query.ndim != 3 or query.shape[0] != rows_in or query.shape[1] != self.n_q_heads \
                or query.shape[2] != self.head_dim:
            raise ValueError("Query must be [total_q, n_q_heads, head_dim] as planned.")
        if query_rows is not None:
            if append is not None:
                raise ValueError("query_rows and append cannot be combined.")
            if query_rows.dtype != torch.int64 or query_rows.ndim != 1 or not query_rows.is_contiguous() \
                    or query_rows.numel() != self.total_q or query_rows.device != self.device:
                raise ValueError("query_rows must be contiguous int64 [total_q] on the plan's device.")
            if query.shape[0] < 1:
                raise ValueError("query_rows needs a query tensor of at least one row.")
        if k_cache.shape != v_cache.shape or k_cache.dtype != query.dtype or v_cache.dtype != query.dtype:
            raise ValueError("Key/value caches must match each other and the query dtype.")
        if k_cache.stride() != v_cache.stride():
            raise ValueError("Key and value caches must share strides.")
        if self.page_size > 0:
            if k_cache.ndim != 4 or k_cache.shape[1] != self.page_size:
                raise ValueError("Paged caches must be [num_pages, page_size, kv_heads, head_dim].")
            if block_table is None or block_table.dtype != torch.int32 or block_table.ndim != 2 \
                    or block_table.shape[0] != self.batch or block_table.device != self.device:
                raise ValueError("block_table must be int32 [batch, width] on the query's device.")
            if block_table.stride(1) != 1 or block_table.shape[1] != self.block_table_stride \
                    or block_table.stride(0) != self.block_table_stride:
                raise ValueError("block_table must be row-contiguous with the planned width.")
            num_pages = k_cache.shape[0]
            row_stride, head_stride = k_cache.stride(1), k_cache.stride(2)
            if k_cache.stride(0) != self.page_size * row_stride:
                raise ValueError("Pages must be laid out back to back.")
        else:
            if k_cache.ndim != 3:
                raise ValueError("Packed caches must be [total_k, kv_heads, head_dim].")
            num_pages = 0
            row_stride, head_stride = k_cache.stride(0), k_cache.stride(1)
        if k_cache.shape[-2] != self.n_kv_heads or k_cache.shape[-1] != self.head_dim or k_cache.stride(-1) != 1:
            raise ValueError("Key/value caches must be [..., n_kv_heads, head_dim] with contiguous head_dim.")
        if query.stride(2) != 1:
            query = query.contiguous()
        out_shape = (self.total_q, self.n_q_heads, self.head_dim)
        if out is None:
            out = torch.empty(out_shape, dtype=query.dtype, device=query.device)
        elif tuple(out.shape) != out_shape or out.dtype != query.dtype or out.stride(2) != 1:
            raise ValueError("out must be [total_q, n_q_heads, head_dim] of the query's dtype.")
        lse = lse_out
        if lse is not None:
            if lse.dtype != torch.float32 or tuple(lse.shape) != (self.n_q_heads, self.total_q) \
                    or not lse.is_contiguous():
                raise ValueError("lse_out must be contiguous float32 [n_q_heads, total_q].")
        elif return_lse:
            lse = torch.empty((self.n_q_heads, self.total_q), dtype=torch.float32, device=query.device)
        scale = 1.0 / math.sqrt(self.head_dim) if scale is None else float(scale)
        hints = (
            self.hints[0] if "decode" in phases else 0,
            self.hints[1] if "chunk" in phases else 0,
            self.hints[2] if "combine" in phases else 0,
        )
        if not self.tuned:
            # The any-head_dim kernel covers every row in one launch and merges in the next:
            # both run in the call that holds the decode phase, or in the chunk phase of a
            # tick without decode rows, never twice for one layer.
            once = "decode" in phases or ("chunk" in phases and self.hints[0] == 0)
            hints = (self.hints[0], self.hints[1], hints[2]) if once else (0, 0, hints[2])
        common = (
            query.data_ptr(), query.stride(0), query.stride(1),
            k_cache.data_ptr(), v_cache.data_ptr(), row_stride, head_stride,
            num_pages, self.page_size,
            None if block_table is None else block_table.data_ptr(), self.block_table_stride,
            self.batch, self.total_q, self.max_q, self.max_k,
            self.n_q_heads, self.n_kv_heads, self.head_dim,
            scale, self.window[0], self.window[1], _SUPPORTED[query.dtype],
            out.data_ptr(), out.stride(0), out.stride(1),
            None if lse is None else lse.data_ptr(),
        )
        if merge is not None:
            if append is not None or query_rows is not None:
                raise ValueError("merge cannot be combined with append or query_rows.")
            if "combine" not in phases or lse is None or not self.tuned:
                raise ValueError("merge needs the combine phase, the lse output and a tuned shape.")
            lo, ll = merge.level_out, merge.level_lse
            n_a = lo.shape[0] if lo.ndim == 3 else -1
            if lo.ndim != 3 or lo.shape[1:] != (self.n_q_heads, self.head_dim) or lo.dtype != query.dtype \
                    or lo.stride(2) != 1 or lo.device != self.device:
                raise ValueError("merge.level_out must be [rows, n_q_heads, head_dim] of the query's dtype.")
            if ll.dtype != torch.float32 or tuple(ll.shape) != (self.n_q_heads, n_a) or not ll.is_contiguous():
                raise ValueError("merge.level_lse must be contiguous float32 [n_q_heads, rows].")
            for name in ("member_seq", "member_of_seq", "part_start", "part_idx"):
                t = getattr(merge, name)
                if t.dtype != torch.int32 or t.ndim != 1 or not t.is_contiguous() or t.device != self.device:
                    raise ValueError(f"merge.{name} must be a contiguous int32 vector on the device.")
            n_members = merge.member_seq.numel()
            if merge.part_start.numel() != n_members + 1 or merge.member_of_seq.numel() != self.batch:
                raise ValueError("merge.part_start needs members + 1 entries and member_of_seq one per sequence.")
            lp = merge.level_plan
            if lp is None:
                code = _capi.lib().hx_varlen_attn_run_merged(
                    *common, lo.data_ptr(), lo.stride(0), lo.stride(1), ll.data_ptr(), n_a,
                    merge.member_seq.data_ptr(), merge.member_of_seq.data_ptr(), n_members,
                    merge.part_start.data_ptr(), merge.part_idx.data_ptr(), merge.part_idx.numel(),
                    *hints, self.ws_ptr, self.ws_bytes, _stream_ptr(query.device))
                _capi.check(code, "hx_varlen_attn_run_merged")
            else:
                if not isinstance(lp, VarlenAttnPlan) or lp.device != self.device or lp.n_q_heads != self.n_q_heads \
                        or lp.n_kv_heads != self.n_kv_heads or lp.head_dim != self.head_dim or lp.total_q != n_a:
                    raise ValueError("merge.level_plan must be the plan of level_out: same device and heads, "
                                     "total_q = level_out rows.")
                lbt, lrows = merge.level_block_table, merge.level_query_rows
                if lbt is None and lrows is not None:
                    raise ValueError("merge.level_query_rows needs merge.level_block_table.")
                if lbt is not None:
                    # The level plan's chunk items run in this call (see MergeParts).
                    if set(phases) != {"decode", "chunk", "combine"}:
                        raise ValueError("a merge that runs the level plan's chunk items needs all three phases.")
                    if lp.hints[0] != 0 or lp.page_size != self.page_size:
                        raise ValueError("merge.level_plan must hold no decode rows and share the page size to "
                                         "run in this call.")
                    if lp.page_size > 0 and (lbt.dtype != torch.int32 or lbt.ndim != 2 or lbt.shape[0] != lp.batch
                                             or lbt.shape[1] != lp.block_table_stride or lbt.stride(1) != 1
                                             or lbt.stride(0) != lp.block_table_stride or lbt.device != self.device):
                        raise ValueError("merge.level_block_table must be the level plan's row-contiguous int32 "
                                         "[batch, width] table on the device.")
                    if lrows is None or lrows.dtype != torch.int64 or lrows.ndim != 1 or not lrows.is_contiguous() \
                            or lrows.numel() != lp.total_q or lrows.device != self.device:
                        raise ValueError("merge.level_query_rows must be contiguous int64 [level rows] on the device.")
                level_chunk = (None, 0, None, 0, 0, -1, -1) if lbt is None else (
                    lbt.data_ptr(), lp.block_table_stride, lrows.data_ptr(), query.shape[0], lp.hints[1],
                    lp.window[0], lp.window[1])
                code = _capi.lib().hx_varlen_attn_run_cascade(
                    *common, lo.data_ptr(), lo.stride(0), lo.stride(1), ll.data_ptr(), n_a,
                    lp.batch, lp.max_q, lp.max_k, lp.hints[2], lp.ws_ptr, lp.ws_bytes, *level_chunk,
                    merge.member_seq.data_ptr(), merge.member_of_seq.data_ptr(), n_members,
                    merge.part_start.data_ptr(), merge.part_idx.data_ptr(), merge.part_idx.numel(),
                    *hints, self.ws_ptr, self.ws_bytes, _stream_ptr(query.device))
                _capi.check(code, "hx_varlen_attn_run_cascade")
        elif query_rows is not None:
            code = _capi.lib().hx_varlen_attn_run_rows(
                *common[:3], query_rows.data_ptr(), query.shape[0], *common[3:], *hints,
                self.ws_ptr, self.ws_bytes, _stream_ptr(query.device))
            _capi.check(code, "hx_varlen_attn_run_rows")
        elif append is None:
            code = _capi.lib().hx_varlen_attn_run(
                *common, *hints, self.ws_ptr, self.ws_bytes, _stream_ptr(query.device))
            _capi.check(code, "hx_varlen_attn_run")
        else:
            k_new, v_new, slots = append
            _check_append(k_cache, v_cache, slots, k_new, v_new)
            if k_new.shape[0] != self.total_q:
                raise ValueError("append rows must match the packed query rows.")
            if not k_cache.is_contiguous() or not v_cache.is_contiguous():
                raise ValueError("KV pools must be contiguous.")
            pool_rows = k_cache.numel() // (self.n_kv_heads * self.head_dim)
            slots = slots.contiguous()
            code = _capi.lib().hx_varlen_attn_append_run(
                *common,
                k_new.data_ptr(), k_new.stride(0), k_new.stride(1),
                v_new.data_ptr(), v_new.stride(0), v_new.stride(1),
                slots.data_ptr(), pool_rows,
                *hints, self.ws_ptr, self.ws_bytes, _stream_ptr(query.device))
            _capi.check(code, "hx_varlen_attn_append_run")
        if CHECK_ERRORS:
            self.check_errors()
            if merge is not None and merge.level_plan is not None:
                merge.level_plan.check_errors()  # its combine records (and chunk items) ran in this call
        return (out, lse) if return_lse else out


def run_overlapped(plan: "VarlenAttnPlan", query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   block_table: torch.Tensor | None, side: torch.cuda.Stream, *, return_lse: bool = False,
                   side_first=None):
    """``plan.run`` with the chunk rows (MFMA-bound) on ``side`` while the decode rows
    (HBM-bound) run on the current stream; the combine runs after both. The new K/V rows
    must already be in the pool. ``side_first`` is an optional callable queued on the
    side stream before the chunk launch (work that must also overlap the decode rows);
    its return value is returned last, and any tensors in it are marked as used by the
    current stream. Falls back to ``plan.run`` when one kind of row is absent, and for
    shapes the any-head_dim kernel serves (it covers every row in one launch)."""
    dec, pf, _ = plan.hints
    has_chunk = pf != 0 and plan.max_q >= 2
    if dec == 0 or (not has_chunk and side_first is None) or not plan.tuned:
        extra = side_first() if side_first is not None else None
        res = plan.run(query, k_cache, v_cache, block_table, return_lse=return_lse)
        return (res, extra) if side_first is not None else res
    main = torch.cuda.current_stream(query.device)
    out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    lse = torch.empty((plan.n_q_heads, plan.total_q), dtype=torch.float32, device=query.device) if return_lse else None
    forked = torch.cuda.Event()
    forked.record(main)
    side.wait_event(forked)
    extra = None
    with torch.cuda.stream(side):
        if side_first is not None:
            extra = side_first()
        if has_chunk:
            plan.run(query, k_cache, v_cache, block_table, out=out, lse_out=lse, phases=("chunk",))
    joined = torch.cuda.Event()
    joined.record(side)
    plan.run(query, k_cache, v_cache, block_table, out=out, lse_out=lse, phases=("decode",))
    main.wait_event(joined)
    if extra is not None:
        for t in (extra if isinstance(extra, tuple) else (extra,)):
            if isinstance(t, torch.Tensor):
                t.record_stream(main)
    plan.run(query, k_cache, v_cache, block_table, out=out, lse_out=lse, phases=("combine",))
    res = (out, lse) if return_lse else out
    return (res, extra) if side_first is not None else res


def varlen_attn(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    cu_seq_q: torch.Tensor,
    cu_seq_k: torch.Tensor | None,
    max_q: int,
    max_k: int,
    is_causal: bool = False,
    return_aux: AuxRequest | None = None,
    *,
    window_size: tuple[int, int] | None = None,
    enable_gqa: bool = False,
    seqused_k: torch.Tensor | None = None,
    block_table: torch.Tensor | None = None,
    num_splits: int | None = None,
    scale: float | None = None,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Drop-in for the paged ``varlen_attn`` call at paged_cache.py:316-329 / :506-519.

    ``query``: ``[total_q, Hq, d]``. With ``block_table`` (int32 ``[B, W]``),
    ``key``/``value`` are pools ``[num_pages, page_size, Hkv, d]`` and sequence b
    has ``seqused_k[b]`` keys (else ``cu_seq_k[b+1]-cu_seq_k[b]``); without it they
    are packed ``[total_k, Hkv, d]`` located by ``cu_seq_k``. ``window_size=(-1, 0)``
    is the bottom-right causal mask. ``num_splits`` is accepted for signature parity:
    the split schedule is fixed by each sequence's length, and the combine order is
    fixed, so results are deterministic for any value.
    """
    del num_splits
    device = _require_gpu(query, key, value, cu_seq_q)
    if query.ndim != 3:
        raise ValueError("query must be [total_q, n_q_heads, head_dim].")
    n_q_heads, head_dim = query.shape[1], query.shape[2]
    n_kv_heads = key.shape[-2]
    if n_q_heads != n_kv_heads and not enable_gqa:
        raise ValueError("Query and KV head counts differ; pass enable_gqa=True.")
    if n_kv_heads < 1 or n_q_heads % n_kv_heads:
        raise ValueError(f"GQA needs n_q_heads ({n_q_heads}) to be a multiple of n_kv_heads ({n_kv_heads}).")
    window = _window(window_size, is_causal)
    paged = block_table is not None
    if paged:
        page_size = key.shape[1]
        bt_stride = block_table.shape[1] if block_table.ndim == 2 else 0
        if block_table.stride(-1) != 1:
            block_table = block_table.contiguous()
        total_k_rows = 0
    else:
        if cu_seq_k is None:
            raise ValueError("Packed keys need cu_seq_k.")
        page_size, bt_stride = 0, 0
        total_k_rows = key.shape[0]
    plan = VarlenAttnPlan(
        cu_seq_q, cu_seq_k, seqused_k,
        total_q=query.shape[0], max_q=max_q, max_k=max_k,
        n_q_heads=n_q_heads, n_kv_heads=n_kv_heads, head_dim=head_dim,
        page_size=page_size, block_table_stride=bt_stride, total_k_rows=total_k_rows,
        window=window,
    )
    want_lse = bool(return_aux is not None and return_aux.lse)
    del device
    return plan.run(query, key, value, block_table, scale=scale, return_lse=want_lse)
