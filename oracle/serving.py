"""The serving operators in 64 bits, sequence by sequence: attention of packed prompts, the
8-bit key/value cache, attention over it. Beside a result stands the bound of its error.

A bound counts roundings: a value rounded to a type is off by at most ``finfo(type).eps / 2`` of itself.
``terms`` of a row is ``sum_j p_j |v_j|`` (the probabilities sum to one): what a relative error of the
probabilities is multiplied by. ``size`` is the largest ``scale * sum_d |q_d k_d|``: what the relative
error of a product is multiplied by to be an absolute error of a score, and so a relative one of a probability.
"""

from __future__ import annotations

import torch
from torch import Tensor

SMALLEST_SCALE = 2.0 ** -100


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def one_sequence(q: Tensor, k: Tensor, v: Tensor, scale: float, causal: bool, p_step: float, q_step: float) -> tuple[Tensor, Tensor]:
    """``q [n, heads, dim]`` over ``k, v [m, kv_heads, dim]``: the result in f64 and the bound of the error of a kernel that
    rounds probabilities by ``p_step`` and queries by ``q_step`` relative to the row's largest."""
    out_dtype = q.dtype
    q, k, v = q.double(), k.double(), v.double()
    n, heads, dim = q.shape
    m, group = k.shape[0], heads // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for i in range(n):
        sees = min(m, i + m - n + 1) if causal else m
        if sees <= 0:
            continue
        scores = torch.einsum("hd,jhd->hj", q[i], k[:sees]) * scale
        p = torch.softmax(scores, 1)
        out[i] = torch.einsum("hj,jhd->hd", p, v[:sees])
        terms = torch.einsum("hj,jhd->hd", p, v[:sees].abs())
        size = (torch.einsum("hd,jhd->hj", q[i].abs(), k[:sees].abs()) * abs(scale)).amax(1)
        lost = (q[i].abs().amax(1) * k[:sees].abs().sum(2).amax(0) * abs(scale)) * q_step
        # f32 sums of dim products and of `sees` terms, the exponential's own error (2^-21), the division
        relative = p_step + 2 * ((dim + 8) * 2.0 ** -24 * size + lost) + 2 * sees * 2.0 ** -24 + 2.0 ** -20
        bound[i] = half_step(out_dtype) * out[i].abs() + relative[:, None] * terms * (1 + half_step(out_dtype)) + 1e-37
    return out, bound


def attention_packed(q: Tensor, k: Tensor, v: Tensor, offsets: list[int], k_offsets: list[int], scale: float, causal: bool,
                     p_step: float) -> tuple[Tensor, Tensor]:
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b in range(len(offsets) - 1):
        rows, keys = slice(offsets[b], offsets[b + 1]), slice(k_offsets[b], k_offsets[b + 1])
        out[rows], bound[rows] = one_sequence(q[rows], k[keys], v[keys], scale, causal, p_step, 0.0)
    return out, bound


def append(codes: Tensor, scales: Tensor, x: Tensor, table: Tensor, lengths: list[int], offsets: list[int]) -> None:
    """New tokens ``x [rows, heads, dim]`` into ``codes [blocks, heads, tokens, dim]`` (V's: a transposed view) and ``scales``."""
    tokens = codes.shape[2]
    for b, length in enumerate(lengths):
        new = x[offsets[b]:offsets[b + 1]].double()
        position = length
        while position < length + new.shape[0]:
            block, first = int(table[b, position // tokens]), position % tokens
            stop = min(tokens, length + new.shape[0] - position + first)
            part = new[position - length:position - length + stop - first].transpose(0, 1)  # [heads, new, dim]
            for head in range(codes.shape[1]):
                values = part[head]
                old = scales[block, head].double() if first else torch.tensor(0.0, dtype=torch.float64)
                if not bool(torch.isfinite(values).all()) or bool(old.isnan()):
                    scales[block, head] = float("nan")
                    codes[block, head, first:stop] = 0
                    continue
                scale = (values.abs().max() / 127).float().double().clamp(min=SMALLEST_SCALE)
                scale = torch.maximum(scale, old)
                if first and scale > old:
                    codes[block, head, :first] = (codes[block, head, :first].double() * old / scale).round().to(torch.int8)
                scales[block, head] = scale.float()
                codes[block, head, first:stop] = (values / scale).round().to(torch.int8)
            position += stop - first


def sequence(codes: Tensor, scales: Tensor, row: Tensor, length: int) -> Tensor:
    """Positions 0 .. length of one sequence, ``[length, heads, dim]`` in f64."""
    tokens = codes.shape[2]
    blocks = row[: -(-length // tokens)].long()
    values = codes[blocks].double() * scales[blocks].double()[:, :, None, None]
    return values.transpose(1, 2).reshape(-1, codes.shape[1], codes.shape[3])[:length]


def attention_cached(q: Tensor, cache: tuple[Tensor, Tensor, Tensor, Tensor], table: Tensor, lengths: list[int], scale: float,
                     p_step: float, q_step: float) -> tuple[Tensor, Tensor]:
    """``q [batch, tokens, heads, dim]``."""
    k_codes, v_codes, k_scales, v_scales = cache
    out, bound = [], []
    for b, length in enumerate(lengths):
        k = sequence(k_codes, k_scales, table[b], length)
        v = sequence(v_codes.transpose(2, 3), v_scales, table[b], length)
        o, e = one_sequence(q[b], k, v, scale, True, p_step, q_step)
        out.append(o)
        bound.append(e)
    return torch.stack(out), torch.stack(bound)
