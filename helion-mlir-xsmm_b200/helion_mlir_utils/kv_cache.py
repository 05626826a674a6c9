"""A key/value cache held in 8 bits and the attention that reads it (no counterpart in the
reference, which has attention over whole operands only).

The cache is four tensors, a :class:`QuantizedCache` or any tuple of the same four:

* ``k_codes`` int8 ``[blocks, heads, tokens, dim]`` and ``v_codes`` int8 ``[blocks, heads, dim, tokens]``
  (V's tokens side by side: the product with the probabilities sums over them);
* ``k_scales``, ``v_scales`` f32 ``[blocks, heads]``: a value is ``code * scale``.

A block holds 16, 32 or 64 tokens; ``dim`` is 64 or 128. Position ``p`` of sequence ``b`` lies in block
``block_table[b, p // tokens]``; who owns which block is the caller's business. Lengths, starts, offsets and the
table are int32 tensors on the device: no call reads them on the host, so all of them can be captured into a CUDA
graph and replayed with other contents. Block numbers outside the cache and positions beyond the table
are not followed: they raise bit 512 of ``native.kernel_status()``, writes skip them and what
reads them answers NaN.

A serving loop: :func:`~helion_mlir_utils.attention_packed` over the prompts and :func:`cache_append` of their keys and
values, then for each token :func:`cache_append` and :func:`attention_cached`; :func:`cache_read` gives a cached
prefix back for ``attention_packed`` of a later chunk of the prompt.
"""

from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch
from torch import Tensor

from helion_mlir_backend import native
from helion_mlir_backend.call_trace import CallExplanation

BLOCK_TOKENS = (16, 32, 64)
HEAD_DIMS = (64, 128)


class QuantizedCache(NamedTuple):
    """Codes and scales of an 8-bit key/value cache; :func:`quantized_cache` allocates one."""

    k_codes: Tensor
    v_codes: Tensor
    k_scales: Tensor
    v_scales: Tensor


def quantized_cache(blocks: int, heads: int, dim: int, block_tokens: int = 64, device: torch.device | str = "cuda") -> QuantizedCache:
    """An empty cache of ``blocks`` blocks for ``heads`` key/value heads. Each head costs ``2 * dim`` bytes a token
    and 8 bytes a block."""
    if blocks < 0 or heads < 1 or dim not in HEAD_DIMS or block_tokens not in BLOCK_TOKENS:
        raise ValueError(f"quantized_cache() expects heads >= 1, dim in {HEAD_DIMS} and block_tokens in {BLOCK_TOKENS}, "
                         f"got {blocks} blocks, heads {heads}, dim {dim}, block_tokens {block_tokens}")
    return QuantizedCache(
        torch.zeros(blocks, heads, block_tokens, dim, dtype=torch.int8, device=device),
        torch.zeros(blocks, heads, dim, block_tokens, dtype=torch.int8, device=device),
        torch.zeros(blocks, heads, dtype=torch.float32, device=device),
        torch.zeros(blocks, heads, dtype=torch.float32, device=device),
    )


_PACK_APPEND = native.packer(native.KvAppendDesc)
_PACK_READ = native.packer(native.KvReadDesc)
_PACK_CACHED = native.packer(native.CachedAttentionDesc)
_DTYPES = {torch.float32: native.F32, torch.bfloat16: native.BF16}


def _describe(cache: tuple[Tensor, Tensor, Tensor, Tensor], name: str) -> tuple[int, ...]:
    """The fields of ``b200_kv_cache``, after the checks of the four tensors."""
    k_codes, v_codes, k_scales, v_scales = cache
    shape = k_codes.shape
    if len(shape) != 4:
        raise ValueError(f"{name}() expects codes [blocks, heads, tokens, dim] and [blocks, heads, dim, tokens], "
                         f"got {tuple(k_codes.shape)} and {tuple(v_codes.shape)}")
    blocks, heads, tokens, dim = shape
    if dim not in HEAD_DIMS or tokens not in BLOCK_TOKENS or heads < 1:
        raise ValueError(f"{name}() expects blocks of {BLOCK_TOKENS} tokens and heads of {HEAD_DIMS}, got codes {tuple(k_codes.shape)}")
    if v_codes.shape != (blocks, heads, dim, tokens) or k_scales.shape != (blocks, heads) or v_scales.shape != (blocks, heads):
        raise ValueError(f"{name}() cache tensors do not match: codes {tuple(k_codes.shape)} and {tuple(v_codes.shape)}, "
                         f"scales {tuple(k_scales.shape)} and {tuple(v_scales.shape)}")
    if not (k_codes.dtype is v_codes.dtype is torch.int8 and k_scales.dtype is v_scales.dtype is torch.float32):
        raise ValueError(f"{name}() expects int8 codes and f32 scales, got {k_codes.dtype}, {v_codes.dtype}, {k_scales.dtype}, {v_scales.dtype}")
    if not (k_codes.is_contiguous() and v_codes.is_contiguous() and k_scales.is_contiguous() and v_scales.is_contiguous()):
        raise ValueError(f"{name}() expects contiguous cache tensors")
    return k_codes.data_ptr(), v_codes.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), blocks, heads, dim, tokens, 0


def _indices(name: str, what: str, t: Tensor, count: int) -> int:
    """The address of an int32 vector of ``count`` values."""
    if t.dtype is not torch.int32 or t.dim() != 1 or t.numel() != count or not t.is_contiguous():
        raise ValueError(f"{name}() expects {what} as a contiguous int32 tensor [{count}], got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _table(name: str, table: Tensor) -> tuple[int, int, int]:
    """Sequences, row stride and width of a block table."""
    if table.dtype is not torch.int32 or table.dim() != 2:
        raise ValueError(f"{name}() expects block_table as an int32 tensor [sequences, blocks], got {table.dtype} {tuple(table.shape)}")
    batch, width = table.shape
    stride, step = table.stride()
    if width > 1 and step != 1:
        raise ValueError(f"{name}() expects block_table with contiguous rows, got strides {table.stride()}")
    if batch > 1 and stride < width:
        raise ValueError(f"{name}() expects block_table rows that do not overlap, got strides {table.stride()}")
    return batch, stride, width


def _aligned_rows(t: Tensor) -> Tensor:
    """``t`` ``[rows, heads, dim]`` if its rows can be read as 16-byte vectors, else a contiguous copy."""
    row, head, dim = t.stride()
    step = 16 // t.element_size()
    if dim == 1 and not (row % step or head % step or t.data_ptr() % 16):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def cache_append(cache: tuple[Tensor, Tensor, Tensor, Tensor], k: Tensor, v: Tensor, block_table: Tensor, lengths: Tensor,
                 offsets: Tensor | None = None) -> None:
    """Write new keys and values behind the ``lengths[b]`` positions that sequence ``b`` holds, in place.

    ``k``, ``v``: bf16 or f32, ``[rows, heads, dim]`` with sequence ``b`` owning the rows ``offsets[b] .. offsets[b + 1]``
    (int32, ``[sequences + 1]``); without ``offsets``, ``[sequences, heads, dim]`` (one token each) or
    ``[sequences, new, heads, dim]``. Views with strides (slices of a fused projection) are read in place.

    Scale of a block and head: ``max(max|x| / 127, 2^-100)`` over the block's tokens; it grows while the block fills and never
    shrinks, and when it grows the older codes become ``rint(code * old / new)``. Codes are rounded to the nearest, ties to
    even. A value that is not finite makes the scale NaN. ``lengths`` is left as it is (the caller adds the
    new tokens); the blocks have to be in the table already. No block may belong to two of the sequences that are written."""
    fields = _describe(cache, "cache_append")
    heads, dim = fields[5], fields[6]
    batch, stride, width = _table("cache_append", block_table)
    code = _DTYPES.get(k.dtype)
    if code is None or k.dtype is not v.dtype or k.shape != v.shape:
        raise ValueError(f"cache_append() expects matching bf16/f32 k and v, got {tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
    shape = k.shape
    if len(shape) == 4 and offsets is None and shape[0] == batch:
        k, v = k.flatten(0, 1), v.flatten(0, 1)
        shape = k.shape
    elif len(shape) != 3 or (offsets is None and shape[0] != batch):
        raise ValueError(f"cache_append() expects k and v [rows, heads, dim] with offsets, or [sequences, heads, dim] or [sequences, new, "
                         f"heads, dim] of {batch} sequences without, got {tuple(k.shape)}")
    if shape[1] != heads or shape[2] != dim:
        raise ValueError(f"cache_append() expects k and v of {heads} heads of {dim}, got {tuple(k.shape)}")
    lengths_ptr = _indices("cache_append", "lengths", lengths, batch)
    offsets_ptr = 0 if offsets is None else _indices("cache_append", "offsets", offsets, batch + 1)
    index = native.index_of(k, v, *cache, block_table, lengths, offsets)
    with native.on_index(index):
        k, v = _aligned_rows(k), _aligned_rows(v)
        (k_row, k_head, _), (v_row, v_head, _) = k.stride(), v.stride()
        result = native.module().b200_kv_append(
            _PACK_APPEND(*fields, code, 0, k.data_ptr(), v.data_ptr(), k_row, k_head, v_row, v_head, block_table.data_ptr(),
                         lengths_ptr, offsets_ptr, stride, width, batch, shape[0]),
            native.raw_stream(index))
    native.check("b200_kv_append", result)


def cache_read(cache: tuple[Tensor, Tensor, Tensor, Tensor], block_table: Tensor, starts: Tensor, lengths: Tensor,
               offsets: Tensor, rows: int, dtype: torch.dtype = torch.bfloat16) -> tuple[Tensor, Tensor]:
    """Positions ``starts[b] ...`` of each sequence as values: ``(k, v)``, each ``[rows, heads, dim]`` in ``dtype`` (bf16 or f32),
    packed: sequence ``b`` fills the rows ``offsets[b] .. offsets[b + 1]``. Positions that the sequence does not
    hold (at or beyond ``lengths[b]``) and rows behind the last sequence are zeros."""
    fields = _describe(cache, "cache_read")
    heads, dim = fields[5], fields[6]
    batch, stride, width = _table("cache_read", block_table)
    code = _DTYPES.get(dtype)
    if code is None or rows < 0:
        raise ValueError(f"cache_read() expects rows >= 0 and dtype bf16/f32, got {rows} and {dtype}")
    starts_ptr, lengths_ptr = _indices("cache_read", "starts", starts, batch), _indices("cache_read", "lengths", lengths, batch)
    offsets_ptr = _indices("cache_read", "offsets", offsets, batch + 1)
    index = native.index_of(*cache, block_table, starts, lengths, offsets)
    with native.on_index(index):
        k = torch.empty(rows, heads, dim, dtype=dtype, device=block_table.device)
        v = torch.empty_like(k)
        result = native.module().b200_kv_read(
            _PACK_READ(*fields, code, 0, k.data_ptr(), v.data_ptr(), block_table.data_ptr(), starts_ptr, lengths_ptr, offsets_ptr,
                       stride, width, batch, rows),
            native.raw_stream(index))
    native.check("b200_kv_read", result)
    return k, v


def _check_cached(q: Tensor, heads: int, dim: int, batch: int) -> tuple[int, int, int]:
    """Element type, tokens and query heads."""
    code, shape = _DTYPES.get(q.dtype), q.shape
    if code is None or len(shape) not in (3, 4) or shape[-1] != dim or shape[-2] % heads:
        raise ValueError(f"attention_cached() expects bf16/f32 q [sequences, heads, {dim}] or [sequences, tokens, heads, {dim}] with "
                         f"heads a multiple of {heads}, got {q.dtype} {tuple(q.shape)}")
    if shape[0] != batch or shape[-2] == 0:
        raise ValueError(f"attention_cached() expects q of {batch} sequences and at least one head, got {tuple(q.shape)}")
    return code, 1 if len(shape) == 3 else shape[1], shape[-2]


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(index: int, heads: int, dim: int, block_tokens: int, width: int, batch: int, tokens: int, q_heads: int) -> int:
    """Scratch of a call on device ``index``, which goes by sizes alone."""
    desc = native.CachedAttentionDesc(cache=native.KvCacheDesc(heads=heads, dim=dim, block_tokens=block_tokens), table_width=width,
                                      batch=batch, tokens=tokens, heads=q_heads)
    return native.module().b200_attention_cached_workspace_bytes(ctypes.byref(desc))


def attention_cached(q: Tensor, cache: tuple[Tensor, Tensor, Tensor, Tensor], block_table: Tensor, lengths: Tensor,
                     scale: float | None = None) -> Tensor:
    """``softmax(scale * q @ k^T) @ v`` over the cached positions; ``scale`` defaults to ``dim ** -0.5``.

    ``q``: bf16 or f32, ``[sequences, heads, dim]`` (one token each) or ``[sequences, tokens, heads, dim]``: the last
    ``tokens`` of the ``lengths[b]`` positions of sequence ``b``, which :func:`cache_append` has written already;
    token ``i`` sees the positions below ``lengths[b] - tokens + i + 1`` (a row that sees none is zeros). Query head ``h`` reads
    key/value head ``h // (heads // kv_heads)``. Result in ``q``'s type and shape."""
    fields = _describe(cache, "attention_cached")
    dim = fields[6]
    batch, stride, width = _table("attention_cached", block_table)
    code, tokens, heads = _check_cached(q, fields[5], dim, batch)
    lengths_ptr = _indices("attention_cached", "lengths", lengths, batch)
    index = native.index_of(q, *cache, block_table, lengths)
    with native.on_index(index):
        if q.stride(-1) != 1:
            q = q.contiguous()
        out = native.empty_like(q)
        steps = q.stride()
        need = _workspace_bytes(index, fields[5], dim, fields[7], width, batch, tokens, heads)
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        result = native.module().b200_attention_cached(
            _PACK_CACHED(*fields, code, dim ** -0.5 if scale is None else scale, q.data_ptr(), out.data_ptr(), steps[0],
                         steps[1] if tokens > 1 else 0, steps[-2], block_table.data_ptr(), lengths_ptr, stride, width, batch,
                         tokens, heads, workspace.data_ptr(), need),
            native.raw_stream(index))
    native.check("b200_attention_cached", result)
    return out


def _explain_cached(q: Tensor, cache: tuple[Tensor, Tensor, Tensor, Tensor], block_table: Tensor, lengths: Tensor,
                    scale: float | None = None) -> CallExplanation:
    fields = _describe(cache, "attention_cached")
    _, tokens, heads = _check_cached(q, fields[5], fields[6], _table("attention_cached", block_table)[0])
    rows = tokens * (heads // fields[5])
    return CallExplanation(True, f"cached_kernel (mma f16, {8 if rows <= 8 else 16} query rows a tile, {rows} rows a head) + cached_join_kernel")


attention_cached.explain = _explain_cached  # type: ignore[attr-defined]
