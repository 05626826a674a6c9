"""Refusals of the serving operators, none of which needs a GPU: the Python checks, and the C ABI's codes."""

from __future__ import annotations

import ctypes
from pathlib import Path
import re

import pytest
import torch

from helion_mlir_backend import native
import helion_mlir_utils as ops

BF16 = torch.bfloat16


def ints(*values: int) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32)


def host_cache(blocks: int = 4, heads: int = 2, dim: int = 64, tokens: int = 16):
    return ops.quantized_cache(blocks, heads, dim, tokens, device="cpu")


def test_packed_refusals() -> None:
    q, k = torch.zeros(6, 4, 64, dtype=BF16), torch.zeros(6, 2, 64, dtype=BF16)
    at = ints(0, 6)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.attention_packed(q, k, k, at)
    for bad in (q[0], torch.zeros(6, 3, 64, dtype=BF16), torch.zeros(6, 4, 32, dtype=BF16)):
        with pytest.raises(ValueError, match="attention_packed"):
            ops.attention_packed(bad, k, k, at)
    with pytest.raises(ValueError, match="do not match"):
        ops.attention_packed(q, k, k[:3], at)
    with pytest.raises(ValueError, match="bf16/f32"):
        ops.attention_packed(q.half(), k.half(), k.half(), at)
    with pytest.raises(ValueError, match="bf16/f32"):
        ops.attention_packed(q, k.float(), k.float(), at)
    with pytest.raises(ValueError, match="heads of 1 to 256"):
        ops.attention_packed(torch.zeros(6, 2, 300), torch.zeros(6, 2, 300), torch.zeros(6, 2, 300), at)
    for offsets in (at.long(), at[None], ints(0, 0, 6, 0, 6)[::2], ints()):
        with pytest.raises(ValueError, match="offsets"):
            ops.attention_packed(q, k, k, offsets)
    with pytest.raises(ValueError, match="k_offsets"):
        ops.attention_packed(q, k, k, at, ints(0, 3, 6))
    with pytest.raises(ValueError, match="needs k_offsets"):
        ops.attention_packed(q, k[:5], k[:5], at)


def test_cache_refusals() -> None:
    for args in ((4, 2, 96), (4, 0, 64), (-1, 2, 64), (4, 2, 64, 48)):
        with pytest.raises(ValueError, match="quantized_cache"):
            ops.quantized_cache(*args, device="cpu")
    cache = host_cache()
    k = torch.zeros(3, 2, 64, dtype=BF16)
    table, lengths = torch.zeros(3, 2, dtype=torch.int32), ints(0, 0, 0)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.cache_append(cache, k, k, table, lengths)
    wrong = [
        (cache[0].float(), *cache[1:]), (cache[0], cache[0], *cache[2:]), (*cache[:2], cache[2][:2], cache[3]),
        (cache[0][:, :, :8], *cache[1:]), (*cache[:3], cache[3].double()), (cache[0][0], *cache[1:]),
        (cache[0], cache[1].transpose(2, 3).contiguous().transpose(2, 3), *cache[2:]),
    ]
    for bad in wrong:
        with pytest.raises(ValueError, match="cache_append"):
            ops.cache_append(bad, k, k, table, lengths)
    for bad_k, bad_v in ((k, k[:2]), (k.half(), k.half()), (k[:, :1], k[:, :1]), (k[:2], k[:2]), (k[0], k[0]), (k, k.float())):
        with pytest.raises(ValueError, match="cache_append"):
            ops.cache_append(cache, bad_k, bad_v, table, lengths)
    for bad in (table.long(), table[0], torch.zeros(2, 3, dtype=torch.int32).T):
        with pytest.raises(ValueError, match="cache_append"):
            ops.cache_append(cache, k, k, bad, lengths)
    with pytest.raises(ValueError, match="lengths"):
        ops.cache_append(cache, k, k, table, ints(0, 0))
    with pytest.raises(ValueError, match="offsets"):
        ops.cache_append(cache, k, k, table, lengths, ints(0, 1, 2))
    with pytest.raises(ValueError, match="heads, dim"):
        ops.cache_append(cache, k[:, None], k[:, None], table, lengths, ints(0, 1, 2, 3))
    with pytest.raises(ValueError, match="cache_read"):
        ops.cache_read(cache, table, lengths, lengths, ints(0, 1, 2, 3), 3, torch.float16)
    with pytest.raises(ValueError, match="cache_read"):
        ops.cache_read(cache, table, lengths, lengths, ints(0, 1, 2, 3), -1)
    with pytest.raises(ValueError, match="offsets"):
        ops.cache_read(cache, table, lengths, lengths, ints(0, 1), 3)
    q = torch.zeros(3, 4, 64, dtype=BF16)
    for bad in (q.half(), q[:2], q[..., :32], q[:, :3], q[0], q[:, :0]):
        with pytest.raises(ValueError, match="attention_cached"):
            ops.attention_cached(bad, cache, table, lengths)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.attention_cached(q, cache, table, lengths)


def test_c_abi_refusals() -> None:
    lib = native.module()
    buf = torch.zeros(4096, dtype=torch.uint8)
    at = (buf.data_ptr() + 15) // 16 * 16

    def packed(**change):
        fields = dict(dtype=native.BF16, causal=1, q=at, k=at, v=at, out=at, q_row=128, q_head=64, k_row=64, k_head=64, v_row=64,
                      v_head=64, rows_q=4, rows_k=4, batch=1, heads=2, kv_heads=1, dim=64, offsets=at, k_offsets=at, scale=1.0)
        fields.update(change)
        return lib.b200_attention_packed(ctypes.byref(native.PackedAttentionDesc(**fields)), None)

    assert lib.b200_attention_packed(None, None) == 6
    assert packed(dtype=7) == 1
    for change in ({"heads": 3, "kv_heads": 2}, {"dim": 0}, {"dim": 257}, {"rows_q": -1}, {"batch": -1}, {"kv_heads": 0},
                   {"heads": 65536, "kv_heads": 1}, {"rows_k": 1 << 31}):
        assert packed(**change) == 2, change
    assert packed(causal=2) == 7 and packed(scale=float("nan")) == 7 and packed(scale=float("inf")) == 7
    assert packed(q=None) == 6 and packed(out=None) == 6 and packed(offsets=None) == 6 and packed(v=None) == 6
    assert packed(q=at + 1) == 4 and packed(offsets=at + 2) == 4
    assert packed(rows_q=0, q=None) == 0

    def cache(**change):
        fields = dict(k_codes=at, v_codes=at, k_scales=at, v_scales=at, blocks=2, heads=2, dim=64, block_tokens=16)
        fields.update(change)
        return native.KvCacheDesc(**fields)

    def append(c, **change):
        fields = dict(cache=c, dtype=native.BF16, k=at, v=at, k_row=128, k_head=64, v_row=128, v_head=64, block_table=at, lengths=at,
                      offsets=at, table_stride=2, table_width=2, batch=2, rows=2)
        fields.update(change)
        return lib.b200_kv_append(ctypes.byref(native.KvAppendDesc(**fields)), None)

    def read(c, **change):
        fields = dict(cache=c, dtype=native.BF16, k_out=at, v_out=at, block_table=at, starts=at, lengths=at, offsets=at, table_stride=2,
                      table_width=2, batch=2, rows=2)
        fields.update(change)
        return lib.b200_kv_read(ctypes.byref(native.KvReadDesc(**fields)), None)

    def attend(c, **change):
        fields = dict(cache=c, dtype=native.BF16, scale=1.0, q=at, out=at, q_batch=256, q_token=256, q_head=64, block_table=at, lengths=at,
                      table_stride=2, table_width=2, batch=2, tokens=1, heads=4)
        fields.update(change)
        return lib.b200_attention_cached(ctypes.byref(native.CachedAttentionDesc(**fields)), None)

    for call in (append, read, attend):
        assert call(cache(), dtype=5) == 1
        for change in ({"dim": 96}, {"block_tokens": 8}, {"block_tokens": 128}, {"heads": 0}, {"blocks": -1}):
            assert call(cache(**change)) == 2, change
        assert call(cache(k_codes=None)) == 6 and call(cache(v_scales=None)) == 6
        assert call(cache(k_codes=at + 8)) == 4
        assert call(cache(), table_stride=1) == 3 and call(cache(), table_width=-1) == 3
        assert call(cache(), batch=-1) == 2
        assert call(cache(), block_table=at + 2) == 4
    assert append(cache(), offsets=None, rows=3) == 2
    assert append(cache(), k_row=129) == 3 and append(cache(), k=at + 2) == 4
    assert append(cache(), k=None) == 6 and append(cache(), lengths=None) == 6
    assert append(cache(), batch=0) == 0 and append(cache(), rows=0) == 0
    assert read(cache(), k_out=None) == 6 and read(cache(), offsets=None) == 6 and read(cache(), v_out=at + 8) == 4
    assert read(cache(), rows=0) == 0
    assert attend(cache(), heads=3) == 2 and attend(cache(), tokens=-1) == 2 and attend(cache(), scale=float("nan")) == 7
    assert attend(cache(), q=None) == 6 and attend(cache(), batch=0) == 0 and attend(cache(), tokens=0) == 0
    for fn in (lib.b200_kv_append, lib.b200_kv_read, lib.b200_attention_cached):
        assert fn(None, None) == 6
    assert lib.b200_attention_cached_workspace_bytes(None) == 0


_STRUCTS = [
    ("b200_packed_attention_desc", native.PackedAttentionDesc), ("b200_kv_cache", native.KvCacheDesc),
    ("b200_kv_append_desc", native.KvAppendDesc), ("b200_kv_read_desc", native.KvReadDesc),
    ("b200_cached_attention_desc", native.CachedAttentionDesc),
]


def test_packed_descriptors_are_the_structures() -> None:
    """The bytes that the operators pass are those of the ctypes mirror with the same values."""
    for _, kind in _STRUCTS:
        def fill(structure, start: int) -> list[int]:
            values = []
            for name, field in structure._fields_:
                if issubclass(field, ctypes.Structure):
                    values += fill(getattr(structure, name), start + len(values))
                else:
                    values.append(start + len(values) + 1)
                    setattr(structure, name, values[-1])
            return values

        structure = kind()
        assert native.packer(kind)(*fill(structure, 0)) == bytes(structure)


@pytest.mark.parametrize("name,struct", _STRUCTS)
def test_struct_layouts_match_the_header(name: str, struct) -> None:
    text = (Path(__file__).resolve().parent.parent / "include" / "b200ops.h").read_text()
    body = text[text.index(f"typedef struct {name} {{") + len(f"typedef struct {name} {{") : text.index(f"}} {name};")]
    fields = []
    for statement in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
        if statement.strip():
            first, *rest = statement.split(",")
            fields += [first.split()[-1].lstrip("*"), *(n.strip().lstrip("*") for n in rest)]
    assert fields == [field for field, _ in struct._fields_]


def test_explanations_need_no_gpu() -> None:
    q, k = torch.zeros(6, 4, 64, dtype=BF16), torch.zeros(6, 2, 64, dtype=BF16)
    assert ops.attention_packed.explain(q, k, k, ints(0, 6)).native
    assert ops.attention_cached.explain(torch.zeros(1, 4, 64), host_cache(), ints(0)[None], ints(0)).native
