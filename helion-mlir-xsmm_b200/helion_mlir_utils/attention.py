"""Softmax attention built on this operator set (an extension of the reference's
30 names: the reference carries the kernel only as a test body,
``tests/harness.py:263-300`` ``_attention`` and ``tests/test_numerics.py:141-158``
``attention``).

``attention(q, k, v, scale)`` computes ``softmax(scale * q @ k^T) @ v`` per head for
``[heads, seq, dim]`` operands. bf16 operands with ``dim`` 64 or 128 run the fused
tensor-core kernel ``b200_attention`` (scores and probabilities never leave the
SM). Everything else (f32, other head sizes) is composed from the operators of
this package: one batched GEMM for the scores, the row softmax, one batched GEMM
with ``v`` -- the scores then pass through HBM once in f32.

``attention_packed`` is the form that prompts need: sequences of different lengths packed
into one tensor, causal, several query heads to a key/value head.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor

from helion_mlir_backend import native
from helion_mlir_backend import output_pool
from helion_mlir_backend.call_trace import CallExplanation
from helion_mlir_backend.call_trace import trace

_FUSED_DIMS = (64, 128)


def _check(q: Tensor, k: Tensor, v: Tensor) -> tuple[int, int, int, int]:
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError(f"attention() expects [heads, seq, dim] operands, got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    heads, seq_q, dim = map(int, q.shape)
    if int(k.shape[0]) != heads or int(k.shape[2]) != dim or tuple(v.shape) != tuple(k.shape):
        raise ValueError(f"attention() operands do not match: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if not (q.dtype == k.dtype == v.dtype) or q.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"attention() requires matching bf16/f32 operands, got {q.dtype}, {k.dtype}, {v.dtype}")
    return heads, seq_q, int(k.shape[1]), dim


def fused(q: Tensor, k: Tensor, v: Tensor, scale: float = 1.0) -> bool:
    """Whether this call takes the fused kernel (else the composed path)."""
    return (q.dtype == torch.bfloat16 and q.dim() == 3 and int(q.shape[2]) in _FUSED_DIMS
            and scale != 0.0 and math.isfinite(scale))


def attention(q: Tensor, k: Tensor, v: Tensor, scale: float | None = None) -> Tensor:
    """``softmax(scale * q @ k^T, dim=-1) @ v`` per head; ``scale`` defaults to
    ``dim ** -0.5``. Result in ``q.dtype``, shape of ``q``."""
    heads, seq_q, seq_k, dim = _check(q, k, v)
    device = native.require_cuda(q, k, v)
    scale = 1.0 / math.sqrt(dim) if scale is None else float(getattr(scale, "value", scale))
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    if fused(q, k, v, scale):
        out = output_pool.empty_like(q)
        with native.on_device(device):
            code = native.module().b200_attention(
                native.BF16, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), heads, seq_q, seq_k, dim,
                scale, native.stream_ptr(device),
            )
        native.check("b200_attention", code)
        trace(f"attention fused {tuple(q.shape)} x {tuple(k.shape)}")
        return out
    return _composed(q, k, v, scale)


def _composed(q: Tensor, k: Tensor, v: Tensor, scale: float) -> Tensor:
    from . import elementwise, normalization
    from .matmul import bmm

    heads, seq_q, dim = map(int, q.shape)
    seq_k = int(k.shape[1])
    if seq_k == 0 or seq_q == 0 or heads == 0:
        return torch.zeros_like(q)
    # scores = (scale * q) @ k^T: the scale rides on the smaller operand
    scaled = elementwise.scalar_mul(q.reshape(heads * seq_q, dim), scale).reshape(heads, seq_q, dim)
    scores = bmm(scaled, k.transpose(1, 2).contiguous(), out_dtype=torch.float32)
    probs = normalization.softmax(scores.reshape(heads * seq_q, seq_k), in_place=True).reshape(heads, seq_q, seq_k)
    trace(f"attention composed {tuple(q.shape)} x {tuple(k.shape)}")
    return bmm(probs.to(q.dtype), v)


def explain_attention(q: Tensor, k: Tensor, v: Tensor, scale: float | None = None) -> str:
    _check(q, k, v)
    if fused(q, k, v):
        return "native: attention_kernel (tcgen05, 128 queries x 128 keys per step, scores in TMEM)"
    return "native: composed bmm + softmax + bmm (scores pass through HBM once in f32)"


attention.explain = explain_attention  # type: ignore[attr-defined]


# ------------------------------------------------------------------------------- packed sequences

_MAX_DIM = 256


_PACK_PACKED = native.packer(native.PackedAttentionDesc)
_DTYPES = {torch.float32: native.F32, torch.bfloat16: native.BF16}


def _check_packed(q: Tensor, k: Tensor, v: Tensor, offsets: Tensor, k_offsets: Tensor) -> int:
    """The element type's code, after the checks of the operands."""
    shape, k_shape, code = q.shape, k.shape, _DTYPES.get(q.dtype)
    if len(shape) != 3 or len(k_shape) != 3 or v.dim() != 3:
        raise ValueError(f"attention_packed() expects [rows, heads, dim] operands, got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    rows, heads, dim = shape
    key_rows, kv_heads, key_dim = k_shape
    if k_shape != v.shape or key_dim != dim or kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise ValueError("attention_packed() operands do not match (the heads of q have to be a multiple of those of k and v): "
                         f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if not 1 <= dim <= _MAX_DIM:
        raise ValueError(f"attention_packed() expects heads of 1 to {_MAX_DIM}, got {tuple(q.shape)}")
    if code is None or not q.dtype is k.dtype is v.dtype:
        raise ValueError(f"attention_packed() requires matching bf16/f32 operands, got {q.dtype}, {k.dtype}, {v.dtype}")
    _check_offsets("offsets", offsets, offsets)
    if k_offsets is not offsets:
        _check_offsets("k_offsets", k_offsets, offsets)
    elif key_rows != rows:
        raise ValueError(f"attention_packed() needs k_offsets where k has other rows than q: {tuple(q.shape)}, {tuple(k.shape)}")
    return code


def _check_offsets(name: str, t: Tensor, like: Tensor) -> None:
    if t.dtype is not torch.int32 or t.dim() != 1 or t.numel() != like.numel() or t.numel() == 0 or not t.is_contiguous():
        raise ValueError(f"attention_packed() expects {name} as a contiguous int32 tensor [sequences + 1], got {t.dtype} {tuple(t.shape)}")


def _tensor_core(dtype: torch.dtype, dim: int, scale: float) -> bool:
    """Whether the tcgen05 kernel takes these operands (else mma tiles of any head size)."""
    return dtype is torch.bfloat16 and dim in _FUSED_DIMS and scale > 0.0


def _for_tma(t: Tensor) -> Tensor:
    """``t`` if a TMA descriptor can hold its strides, else a contiguous copy."""
    row, head, dim = t.stride()
    if dim == 1 and row > 0 and head > 0 and not (row % 8 or head % 8 or t.data_ptr() % 16):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def attention_packed(q: Tensor, k: Tensor, v: Tensor, offsets: Tensor, k_offsets: Tensor | None = None,
                     scale: float | None = None, causal: bool = True) -> Tensor:
    """Attention of packed sequences: ``softmax(scale * q @ k^T) @ v`` of each sequence's queries over its own keys.

    ``q``: ``[rows, heads, dim]``, ``k``, ``v``: ``[key rows, kv_heads, dim]``, bf16 or f32, ``dim`` up to 256; views with
    strides (slices of a fused projection) are read in place. Query head ``h`` reads key/value head
    ``h // (heads // kv_heads)``. ``offsets``, ``k_offsets`` (int32 on the device, ``[sequences + 1]``): sequence ``b`` owns the
    rows ``offsets[b] .. offsets[b + 1]``; ``k_offsets`` defaults to ``offsets`` (a prompt over itself) and differs where a part of
    the keys was computed before. ``causal``: the queries are the last positions of the keys, row ``i`` of ``n`` sees
    key ``j`` of ``m`` if ``j <= i + m - n``. A row that sees no key is zeros, and so are rows behind the last
    sequence. What a row does not see does not reach it, infinities and NaN included. ``scale`` defaults to ``dim ** -0.5``.

    The offsets are not read on the host: a captured call can be replayed with other lengths of the same total. Offsets
    that decrease or leave the tensors raise bit 256 of ``native.kernel_status()`` and leave their rows unwritten."""
    if k_offsets is None:
        k_offsets = offsets
    code = _check_packed(q, k, v, offsets, k_offsets)
    index = native.index_of(q, k, v, offsets, k_offsets)
    rows, heads, dim = q.shape
    key_rows, kv_heads, _ = k.shape
    scale = dim ** -0.5 if scale is None else float(scale)
    with native.on_index(index):
        if _tensor_core(q.dtype, dim, scale):
            q, k, v = _for_tma(q), _for_tma(k), _for_tma(v)
        elif dim > 1:
            q, k, v = (t if t.stride(2) == 1 else t.contiguous() for t in (q, k, v))
        out = native.empty_like(q)
        (q_row, q_head, _), (k_row, k_head, _), (v_row, v_head, _) = q.stride(), k.stride(), v.stride()
        result = native.module().b200_attention_packed(
            _PACK_PACKED(code, bool(causal), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), q_row, q_head, k_row, k_head,
                         v_row, v_head, rows, key_rows, offsets.numel() - 1, heads, kv_heads, dim, offsets.data_ptr(),
                         k_offsets.data_ptr(), scale, 0),
            native.raw_stream(index))
    native.check("b200_attention_packed", result)
    return out


def _explain_packed(q: Tensor, k: Tensor, v: Tensor, offsets: Tensor, k_offsets: Tensor | None = None,
                    scale: float | None = None, causal: bool = True) -> CallExplanation:
    _check_packed(q, k, v, offsets, offsets if k_offsets is None else k_offsets)
    if _tensor_core(q.dtype, q.shape[2], 1.0 if scale is None else scale):
        return CallExplanation(True, "packed_umma_kernel (tcgen05, two tiles of 128 queries x 128 keys per step, scores in TMEM)")
    return CallExplanation(True, "packed_mma_kernel (mma bf16, f32 values in three pieces, 64 queries a CTA)")


attention_packed.explain = _explain_packed  # type: ignore[attr-defined]
