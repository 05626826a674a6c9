"""Packed prompt attention and the 8-bit key/value cache on the device against the oracle in
64 bits, element by element within bounds that count roundings (oracle/serving.py)."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import serving as ref

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def ops(built_library):
    import helion_mlir_utils

    return helion_mlir_utils


@pytest.fixture(autouse=True)
def status_is_clean(ops):
    from helion_mlir_backend import native

    native.kernel_status()
    yield
    assert native.kernel_status() == 0


def ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def offsets_of(counts: list[int]) -> list[int]:
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def within(actual: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    actual = actual.cpu().double()
    assert actual.shape == want.shape, what
    assert torch.equal(actual.isnan(), want.isnan()), f"{what}: NaN elsewhere"
    off = ((actual - want).abs() - bound).nan_to_num(0.0)
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 0, f"{what}: {worst:.3e} beyond the bound at {int(off.argmax())}"


# ------------------------------------------------------------------------------------------------ packed prompts


def packed_operands(dtype, dim: int, heads: int, kv_heads: int, rows: int, key_rows: int, seed: int):
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn(rows, heads, dim, generator=gen).to(dtype)
    k = torch.randn(key_rows, kv_heads, dim, generator=gen).to(dtype)
    v = torch.randn(key_rows, kv_heads, dim, generator=gen).to(dtype)
    return q, k, v


def p_step(dtype) -> float:
    # bf16: the rounding of P, and a cubic in place of some exponentials, 8.6e-5 of a term and of the sum
    return ref.half_step(BF16) + 1.8e-4 if dtype == BF16 else 0.0


def check_packed(ops, dtype, dim, heads, kv_heads, new, keys, causal=True, scale=None, seed=0) -> None:
    at, k_at = offsets_of(new), offsets_of(keys)
    q, k, v = packed_operands(dtype, dim, heads, kv_heads, at[-1], k_at[-1], seed + dim)
    want, bound = ref.attention_packed(q, k, v, at, k_at, dim ** -0.5 if scale is None else scale, causal, p_step(dtype))
    out = ops.attention_packed(q.cuda(), k.cuda(), v.cuda(), ints(at), ints(k_at), scale, causal)
    assert out.dtype == dtype
    within(out, want, bound, f"{dtype} {dim} {new} {keys} {causal}")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize(
    "new,keys",
    [
        ([1], [1]),
        ([1], [300]),
        ([127, 128, 129], [127, 128, 129]),
        ([64, 0, 5, 200], [64, 0, 5, 200]),
        ([3, 130, 60], [140, 131, 700]),  # a part of the keys came before
        ([150, 20, 40], [17, 0, 40]),  # rows that see nothing, and a sequence without keys
        ([300], [300]),
        ([1] * 40, [1] * 40),  # more sequences than a warp has lanes
    ],
)
def test_packed_lengths(ops, dtype, dim: int, new, keys) -> None:
    check_packed(ops, dtype, dim, 4, 2, new, keys)
    check_packed(ops, dtype, dim, 4, 2, new, keys, causal=False)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [1, 17, 40, 80, 96, 200, 256])
def test_packed_other_head_sizes(ops, dtype, dim: int) -> None:
    check_packed(ops, dtype, dim, 3, 3, [70, 1, 66], [70, 9, 66])
    check_packed(ops, dtype, dim, 2, 1, [33], [65], causal=False)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 1), (6, 2), (5, 5)])
def test_packed_head_groups(ops, heads: int, kv_heads: int) -> None:
    for dtype in (BF16, F32):
        check_packed(ops, dtype, 64, heads, kv_heads, [130, 7], [130, 7])
        check_packed(ops, dtype, 128, heads, kv_heads, [50, 137], [180, 137])


@pytest.mark.parametrize("scale", [1.0, 0.0, -0.2, 1e-6])
def test_packed_scales(ops, scale: float) -> None:
    for dtype in (BF16, F32):
        check_packed(ops, dtype, 64, 2, 1, [150], [200], scale=scale)


def test_packed_many_sequences_and_long_one(ops) -> None:
    check_packed(ops, BF16, 128, 2, 1, [17 * (i % 5) for i in range(70)], [17 * (i % 5) + i % 3 for i in range(70)])
    check_packed(ops, BF16, 64, 2, 1, [1100], [1400], seed=3)


def test_packed_growing_scores(ops) -> None:
    """Every block of keys scores far above the ones before: the running maximum moves all the time."""
    n, dim = 700, 128
    q, k, v = packed_operands(BF16, dim, 2, 1, n, n, 5)
    k = (k.float() * torch.linspace(0.1, 9.0, n)[:, None, None]).to(BF16)
    want, bound = ref.attention_packed(q, k, v, [0, n], [0, n], 1.0, True, p_step(BF16))
    within(ops.attention_packed(q.cuda(), k.cuda(), v.cuda(), ints([0, n]), scale=1.0), want, bound, "growing scores")


def test_packed_strided_views(ops) -> None:
    """Slices of one fused projection, in both orders of rows and heads; an unaligned view too."""
    heads, kv_heads, at = 4, 2, [0, 90, 260]
    for dtype in (BF16, F32):
        for dim in (64, 128, 40):
            fused = torch.randn(260, (heads + 2 * kv_heads) * dim, generator=torch.Generator().manual_seed(dim)).to(dtype)
            parts = fused.split([heads * dim, kv_heads * dim, kv_heads * dim], 1)
            q, k, v = (p.unflatten(1, (-1, dim)) for p in parts)
            want, bound = ref.attention_packed(q, k, v, at, at, dim ** -0.5, True, p_step(dtype))
            moved = [p.unflatten(1, (-1, dim)) for p in fused.cuda().split([heads * dim, kv_heads * dim, kv_heads * dim], 1)]
            within(ops.attention_packed(*moved, ints(at)), want, bound, f"fused {dtype} {dim}")
            swapped = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in moved]  # heads outermost
            within(ops.attention_packed(*swapped, ints(at)), want, bound, f"heads first {dtype} {dim}")
            shifted = [torch.zeros(t.numel() + 1, dtype=dtype, device="cuda")[1:].view(t.shape).copy_(t) for t in moved]
            within(ops.attention_packed(*shifted, ints(at)), want, bound, f"unaligned {dtype} {dim}")
            last = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in moved]  # dim not contiguous
            within(ops.attention_packed(*last, ints(at)), want, bound, f"dim strided {dtype} {dim}")


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (F32, 64), (BF16, 48)])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_packed_values_that_a_row_does_not_see(ops, dtype, dim: int, bad: float) -> None:
    """Infinities and NaN in keys and values of later positions and of other sequences reach no row."""
    new = [40, 150, 30]
    at = offsets_of(new)
    q, k, v = packed_operands(dtype, dim, 2, 1, at[-1], at[-1], 8)
    want, bound = ref.attention_packed(q, k, v, at, at, dim ** -0.5, True, p_step(dtype))
    k, v = k.clone(), v.clone()
    k[at[1] + 140:at[2]], v[at[1] + 140:at[2]] = bad, bad  # the end of sequence 1: rows before it are as they were
    k[at[2] + 5, 0, 3], v[at[2] + 5, 0, 3] = bad, bad
    out = ops.attention_packed(q.cuda(), k.cuda(), v.cuda(), ints(at)).cpu()
    clean = torch.cat([torch.arange(at[1] + 140), torch.arange(at[2], at[2] + 5)])
    within(out[clean], want[clean], bound[clean], f"masked {bad}")
    assert not torch.isfinite(out[at[1] + 140:at[2]]).any()
    assert not torch.isfinite(out[at[2] + 5:, :, 3]).any()
    # no mask: the other sequences alone are hidden
    v[at[1]:at[2]] = bad
    want, bound = ref.attention_packed(q, k, v, at, at, dim ** -0.5, False, p_step(dtype))
    out = ops.attention_packed(q.cuda(), k.cuda(), v.cuda(), ints(at), causal=False).cpu()
    within(out[:at[1]], want[:at[1]], bound[:at[1]], f"another sequence's {bad}")


def test_packed_unseen_values_may_be_huge(ops) -> None:
    """Masked positions with the largest finite values: their probability is zero, not merely tiny."""
    for dtype in (BF16, F32):
        q, k, v = packed_operands(dtype, 128, 2, 1, 200, 200, 4)
        want, bound = ref.attention_packed(q, k, v, [0, 150], [0, 150], 128 ** -0.5, True, p_step(dtype))
        v[140:] = 3.0e38
        out = ops.attention_packed(q.cuda(), k.cuda(), v.cuda(), ints([0, 150]))[:140].cpu()
        within(out, want[:140], bound[:140], f"huge {dtype}")


def test_packed_queries_that_are_not_finite(ops) -> None:
    """A query with a NaN or an infinity answers NaN; the rows beside it in its tile do not notice."""
    for dtype, dim in ((BF16, 128), (F32, 64), (BF16, 40)):
        q, k, v = packed_operands(dtype, dim, 2, 1, 200, 200, 6)
        want, bound = ref.attention_packed(q, k, v, [0, 200], [0, 200], dim ** -0.5, True, p_step(dtype))
        q[70, 1, 3], q[130, 0, 0] = NAN, INF
        out = ops.attention_packed(q.cuda(), k.cuda(), v.cuda(), ints([0, 200])).cpu()
        hit = torch.zeros(200, 2, dtype=torch.bool)
        hit[70, 1] = hit[130, 0] = True
        assert out[hit].isnan().all()
        within(out[~hit], want[~hit], bound[~hit], f"{dtype} {dim}")


def test_packed_rows_behind_the_last_sequence(ops) -> None:
    for dtype, dim in ((BF16, 128), (F32, 64)):
        q, k, v = packed_operands(dtype, dim, 3, 1, 500, 500, 2)
        k[310:], v[310:], q[310:] = NAN, NAN, NAN
        at = [0, 130, 310]
        want, bound = ref.attention_packed(q, k, v, at, at, dim ** -0.5, True, p_step(dtype))
        filler = torch.full((500, 3, dim), NAN, dtype=dtype, device="cuda")  # memory that the result may reuse
        del filler
        out = ops.attention_packed(q.cuda(), k.cuda(), v.cuda(), ints(at))
        within(out, want, bound, "padded batch")
        assert not out[310:].any()
        assert not ops.attention_packed(q.cuda(), k.cuda(), v.cuda(), ints([0])).any()  # no sequence at all


def test_packed_empty(ops) -> None:
    none = torch.zeros(0, 2, 64, dtype=BF16, device="cuda")
    some = torch.ones(5, 2, 64, dtype=BF16, device="cuda")
    assert ops.attention_packed(none, some, some, ints([0, 0]), ints([0, 5])).shape == (0, 2, 64)
    assert not ops.attention_packed(some, none, none, ints([0, 5]), ints([0, 0])).any()


def test_packed_bad_offsets_raise_a_status_bit(ops) -> None:
    from helion_mlir_backend import native

    x = torch.ones(40, 2, 64, dtype=BF16, device="cuda")
    for dtype in (BF16, F32):
        t = x.to(dtype)
        for bad in ([0, 20, 10, 40], [0, 41], [-1, 40]):
            ops.attention_packed(t, t, t, ints(bad))
            assert native.kernel_status() == 256, bad
        out = ops.attention_packed(t, t, t, ints([0, 20, 40]), ints([0, 20, 90]))
        assert native.kernel_status() == 256
        assert (out[:20].float() - 1).abs().max() <= 2.0 ** -8  # the good sequence is served


def test_packed_streams_graphs_and_replays(ops) -> None:
    at = [0, 100, 333]
    q, k, v = packed_operands(BF16, 128, 4, 2, 333, 333, 11)
    q, k, v = q.cuda(), k.cuda(), v.cuda()
    offsets = ints(at)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = ops.attention_packed(q, k, v, offsets)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = ops.attention_packed(q, k, v, offsets)
    torch.cuda.current_stream().wait_stream(side)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    offsets.copy_(ints([0, 290, 333]))  # other lengths, the same total
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.attention_packed(q, k, v, offsets))
    want, bound = ref.attention_packed(q.cpu(), k.cpu(), v.cpu(), [0, 290, 333], [0, 290, 333], 128 ** -0.5, True, p_step(BF16))
    within(out, want, bound, "replayed")


# ------------------------------------------------------------------------------------------------ the cache


def filled_cache(blocks: int, heads: int, dim: int, tokens: int, seed: int):
    """A cache of arbitrary codes and scales, on the host."""
    gen = torch.Generator().manual_seed(seed)
    return (
        torch.randint(-127, 128, (blocks, heads, tokens, dim), generator=gen, dtype=torch.int8),
        torch.randint(-127, 128, (blocks, heads, dim, tokens), generator=gen, dtype=torch.int8),
        torch.rand(blocks, heads, generator=gen) * 0.03 + 0.001,
        torch.rand(blocks, heads, generator=gen) * 0.03 + 0.001,
    )


def table_for(lengths: list[int], tokens: int, seed: int, spare: int = 1) -> tuple[torch.Tensor, int]:
    """Blocks of each sequence, anywhere in the cache; the entries that no position needs point outside it."""
    each = [-(-n // tokens) for n in lengths]
    total = sum(each) + spare
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(lengths), max([1, *each])), 2 ** 31 - 1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(each):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total


def host_copy(cache):
    return tuple(t.clone() for t in cache)


def check_append(ops, dtype, heads, dim, tokens, before, new, x_scale=1.0, use_offsets=True, seed=0):
    after = [a + b for a, b in zip(before, new)]
    table, total = table_for(after, tokens, seed)
    cache = filled_cache(total, heads, dim, tokens, seed + 1)
    gen = torch.Generator().manual_seed(seed + 2)
    at = offsets_of(new)
    k = (torch.randn(at[-1], heads, dim, generator=gen) * x_scale).to(dtype)
    v = (torch.randn(at[-1], heads, dim, generator=gen) * x_scale).to(dtype)
    want = host_copy(cache)
    ref.append(want[0], want[2], k, table, before, at)
    ref.append(want[1].transpose(2, 3), want[3], v, table, before, at)
    moved = tuple(t.cuda() for t in cache)
    if use_offsets:
        ops.cache_append(moved, k.cuda(), v.cuda(), table.cuda(), ints(before), ints(at))
    else:
        n = new[0]
        shape = (len(new), heads, dim) if n == 1 else (len(new), n, heads, dim)
        ops.cache_append(moved, k.cuda().view(shape), v.cuda().view(shape), table.cuda(), ints(before))
    for name, got, expected in zip(("k_codes", "v_codes", "k_scales", "v_scales"), moved, want):
        assert torch.equal(got.cpu(), expected), f"{name}: {dtype} {tokens} {before} {new}"  # whole numbers and whole scales: bit for bit
    return moved, table, after


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens", [16, 32, 64])
def test_append(ops, dtype, dim: int, tokens: int) -> None:
    check_append(ops, dtype, 2, dim, tokens, [0, 5, tokens, 3 * tokens - 1, 0], [1, 2 * tokens, 7, 2, 0])
    check_append(ops, dtype, 1, dim, tokens, [0], [5 * tokens + 3], x_scale=1e-3)
    check_append(ops, dtype, 3, dim, tokens, [1, 0, tokens - 1, 9], [1, 1, 1, 1], use_offsets=False)
    check_append(ops, dtype, 3, dim, tokens, [1, 0, tokens - 1], [3, 3, 3], use_offsets=False)
    check_append(ops, dtype, 1, dim, tokens, [11] * 40, [1 + i % 3 for i in range(40)], x_scale=4.0, seed=7)  # scales grow


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_append_uneven_and_padded(ops, dtype) -> None:
    """One long prompt among sequences that get nothing (few tokens on average), and rows of no sequence."""
    check_append(ops, dtype, 2, 128, 16, [3] * 30, [0] * 17 + [90] + [0] * 12)
    check_append(ops, dtype, 2, 64, 64, [60, 1, 64], [9, 0, 2], x_scale=0.01)
    cache = ops.quantized_cache(4, 2, 64, 16)
    x = torch.randn(50, 2, 64, generator=torch.Generator().manual_seed(1)).to(dtype)
    x[20:] = NAN  # padding behind the last sequence
    ops.cache_append(cache, x.cuda(), x.cuda(), ints([[0, 1], [2, 3]]), ints([0, 0]), ints([0, 5, 20]))
    assert torch.isfinite(cache.k_scales).all() and torch.isfinite(cache.v_scales).all()
    k, _ = ops.cache_read(cache, ints([[0, 1], [2, 3]]), ints([0, 0]), ints([5, 15]), ints([0, 5, 20]), 20, F32)
    step = x[:20].abs().amax().item() / 127
    assert (k.cpu() - x[:20].float()).abs().max() <= 0.5 * step * 1.001


def test_append_ties_zeros_and_extremes(ops) -> None:
    """Quotients that end in one half go to the even code; a block of zeros; the largest and smallest f32 values."""
    tokens, dim = 16, 64
    for dtype in (BF16, F32):
        for top in (127.0, 127.0 * 2 ** 60, 127.0 * 2.0 ** -90, 1e-35, 3.0e38, 0.0):
            cache = tuple(t.cuda() for t in filled_cache(2, 1, dim, tokens, 4))
            x = torch.zeros(16, 1, dim)
            x[0, 0, 0] = top
            x[1, 0, :] = (torch.arange(dim) + 0.5) * (top / 127)  # 0.5, 1.5, ... steps
            x[2, 0, :] = -(torch.arange(dim) + 0.5) * (top / 127)
            x = x.to(dtype)
            want = host_copy(tuple(t.cpu() for t in cache))
            table = torch.tensor([[1]], dtype=torch.int32)
            ref.append(want[0], want[2], x, table, [0], [0, 16])
            ref.append(want[1].transpose(2, 3), want[3], x, table, [0], [0, 16])
            ops.cache_append(cache, x.cuda(), x.cuda(), table.cuda(), ints([0]), ints([0, 16]))
            for got, expected in zip(cache, want):
                assert torch.equal(got.cpu(), expected), (dtype, top)


def test_append_not_finite(ops) -> None:
    """NaN and infinities make their block's scale NaN, for the rest of the block's use, and no other."""
    for bad in (NAN, INF, -INF):
        cache = ops.quantized_cache(4, 2, 64, 16)
        table, x = ints([[2, 0, 1, 3]]), torch.randn(40, 2, 64, generator=torch.Generator().manual_seed(1)).to(BF16)
        x[20, 1, 5] = bad
        ops.cache_append(cache, x.cuda(), x.cuda(), table, ints([0]), ints([0, 40]))
        for scales in (cache.k_scales, cache.v_scales):
            assert torch.equal(scales.cpu().isnan(), torch.tensor([[0, 1], [0, 0], [0, 0], [0, 0]]).bool())
        ops.cache_append(cache, x[:1].cuda(), x[:1].cuda(), table, ints([40]))
        k, _ = ops.cache_read(cache, table, ints([0]), ints([41]), ints([0, 41]), 41, F32)
        assert torch.equal(k.isnan().any(2).cpu().nonzero()[:, 0].unique(), torch.arange(16, 32))
        # a value that is not finite behind older tokens, then a finite one
        ops.cache_append(cache, x[20:21].cuda(), x[20:21].cuda(), table, ints([41]))
        ops.cache_append(cache, x[:1].cuda(), x[:1].cuda(), table, ints([42]))
        assert cache.k_scales[1, 1].isnan() and not cache.k_scales[1, 0].isnan()
        # the block's next use starts anew
        ops.cache_append(cache, x[:16].cuda(), x[:16].cuda(), ints([[1]]), ints([0]), ints([0, 16]))
        assert torch.isfinite(cache.k_scales).sum() == 7


def test_append_strided_views(ops) -> None:
    heads, dim, rows = 2, 64, 50
    fused = torch.randn(rows, 3 * heads * dim, generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
    _, k, v = (p.unflatten(1, (heads, dim)) for p in fused.chunk(3, 1))
    table = ints([[3, 1, 0, 2]])
    plain, strided = ops.quantized_cache(4, heads, dim, 16), ops.quantized_cache(4, heads, dim, 16)
    ops.cache_append(plain, k.contiguous(), v.contiguous(), table, ints([0]), ints([0, rows]))
    ops.cache_append(strided, k, v, table, ints([0]), ints([0, rows]))
    for a, b in zip(plain, strided):
        assert torch.equal(a, b)
    odd = torch.zeros(rows * heads * dim + 1, dtype=BF16, device="cuda")[1:].view(rows, heads, dim).copy_(k)
    ops.cache_append(strided, odd, v.transpose(1, 2).contiguous().transpose(1, 2), table, ints([0]), ints([0, rows]))
    for a, b in zip(plain, strided):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens", [16, 32, 64])
def test_read(ops, dtype, dim: int, tokens: int) -> None:
    lengths, starts = [1, 130, 0, 64, 33], [0, 7, 0, 63, 32]
    table, total = table_for(lengths, tokens, 5)
    cache = filled_cache(total, 3, dim, tokens, 6)
    counts = [n - s for n, s in zip(lengths, starts)]
    counts[3] += 5  # positions that the sequence does not hold
    at = offsets_of(counts)
    rows = at[-1] + 70  # and rows of no sequence
    want = [torch.zeros(rows, 3, dim, dtype=torch.float64) for _ in range(2)]
    for b, n in enumerate(lengths):
        for which, (codes, scales) in enumerate(((cache[0], cache[2]), (cache[1].transpose(2, 3), cache[3]))):
            want[which][at[b]:at[b] + n - starts[b]] = ref.sequence(codes, scales, table[b], n)[starts[b]:]
    moved = tuple(t.cuda() for t in cache)
    got = ops.cache_read(moved, table.cuda(), ints(starts), ints(lengths), ints(at), rows, dtype)
    for name, a, b in zip("kv", got, want):
        within(a, b, b.abs() * (ref.half_step(dtype) + 2.0 ** -24), name)  # one product in f32, one rounding
    empty = ops.cache_read(moved, table.cuda(), ints(starts), ints(lengths), ints([0] * 6), 0, dtype)
    assert empty[0].shape == (0, 3, dim)


# ------------------------------------------------------------------------------------------------ attention over the cache


def steps(dtype) -> tuple[float, float]:
    """Rounding of the probabilities and of the queries by a kernel that multiplies f16 pieces: one piece of 11 bits for
    bf16 operands (whose 8 bits fit, down to 2^-24 of the row's largest), two pieces for f32."""
    return (2.0 ** -11, 2.0 ** -24) if dtype == BF16 else (2.0 ** -21, 2.0 ** -21)


def check_cached(ops, dtype, dim, heads, kv_heads, tokens, lengths, n=1, scale=None, seed=0, squeeze=True):
    table, total = table_for(lengths, tokens, seed)
    cache = filled_cache(total, kv_heads, dim, tokens, seed + 1)
    q = torch.randn(len(lengths), n, heads, dim, generator=torch.Generator().manual_seed(seed + 2)).to(dtype)
    want, bound = ref.attention_cached(q, cache, table, lengths, dim ** -0.5 if scale is None else scale, *steps(dtype))
    arg = q[:, 0] if n == 1 and squeeze else q
    out = ops.attention_cached(arg.cuda(), tuple(t.cuda() for t in cache), table.cuda(), ints(lengths), scale)
    assert out.dtype == dtype and out.shape == arg.shape
    within(out.reshape(q.shape), want, bound, f"{dtype} {dim} {heads}/{kv_heads} {tokens} {lengths} {n}")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens", [16, 32, 64])
def test_cached_lengths(ops, dtype, dim: int, tokens: int) -> None:
    check_cached(ops, dtype, dim, 4, 2, tokens, [1])
    check_cached(ops, dtype, dim, 4, 2, tokens, [0, 63, 64, 65, 1, 200, 0], seed=1)
    check_cached(ops, dtype, dim, 8, 1, tokens, [1000, 3], seed=2)
    check_cached(ops, dtype, dim, 2, 2, tokens, [17] * 40, seed=3)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (7, 1), (10, 2), (16, 1), (24, 2), (40, 1), (64, 1)])
def test_cached_head_groups(ops, dtype, heads: int, kv_heads: int) -> None:
    check_cached(ops, dtype, 64, heads, kv_heads, 16, [100, 0, 129])
    check_cached(ops, dtype, 128, heads, kv_heads, 64, [100, 0, 129])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [1, 2, 5, 9, 40])
def test_cached_several_tokens(ops, dtype, n: int) -> None:
    """Causal among the new tokens; sequences shorter than the tokens asked for have rows that see nothing."""
    check_cached(ops, dtype, 128, 6, 2, 32, [n, 90, n + 1, max(n - 2, 0), 0], n=n, squeeze=False)
    check_cached(ops, dtype, 64, 4, 4, 16, [130, 64], n=n, squeeze=False, seed=4)


@pytest.mark.parametrize("scale", [1.0, 0.0, -0.3])
def test_cached_scales(ops, scale: float) -> None:
    for dtype in (BF16, F32):
        check_cached(ops, dtype, 64, 4, 1, 32, [150, 70], scale=scale)


def test_cached_long(ops) -> None:
    """Many splits of one long sequence, and a batch of uneven ones that share the work."""
    check_cached(ops, BF16, 128, 4, 1, 64, [20000], seed=1)
    check_cached(ops, F32, 64, 2, 1, 16, [7001], seed=2)
    check_cached(ops, BF16, 64, 2, 1, 32, [6000, 10, 0, 333, 2500, 1] * 2, seed=3)


def test_blocks_beyond_32_bits(ops) -> None:
    """Codes of the last blocks of a cache of 5 GB: offsets pass 2^31."""
    heads, dim, tokens, blocks, lengths = 8, 128, 64, 40000, [150]
    cache = ops.quantized_cache(blocks, heads, dim, tokens)
    assert cache.k_codes.numel() > 2 ** 31
    table = torch.tensor([[blocks - 1, 7, blocks - 2]], dtype=torch.int32)
    small = ops.quantized_cache(3, heads, dim, tokens)
    near = torch.tensor([[0, 1, 2]], dtype=torch.int32)
    x = torch.randn(2, 150, heads, dim, generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    q = torch.randn(1, 16, dim, generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
    answers = []
    for c, t in ((cache, table), (small, near)):
        ops.cache_append(c, x[0, :149], x[1, :149], t.cuda(), ints([0]), ints([0, 149]))
        ops.cache_append(c, x[0, 149:], x[1, 149:], t.cuda(), ints([149]))
        answers.append((ops.attention_cached(q, c, t.cuda(), ints(lengths)),
                        *ops.cache_read(c, t.cuda(), ints([0]), ints(lengths), ints([0, 150]), 150)))
    for far, close in zip(*answers):
        assert torch.equal(far, close)
    assert torch.equal(cache.v_codes[blocks - 1], small.v_codes[0])


def test_cached_growing_scores_and_uneven_scales(ops) -> None:
    """Later blocks score far above earlier ones, and their values are of quite different sizes."""
    lengths, tokens, dim = [900], 16, 128
    table, total = table_for(lengths, tokens, 1)
    k_codes, v_codes, k_scales, v_scales = filled_cache(total, 1, dim, tokens, 2)
    order = table[0, :57].long()
    k_scales[order, 0] = torch.linspace(0.001, 0.05, 57)
    v_scales[order, 0] = 10.0 ** (torch.arange(57) % 9 - 4).float()
    v_codes[order[4]] = 0
    v_scales[order[4], 0] = 2.0 ** -100  # what a block of zeros holds
    q = torch.randn(1, 1, 4, dim, generator=torch.Generator().manual_seed(3)).to(BF16)
    cache = (k_codes, v_codes, k_scales, v_scales)
    want, bound = ref.attention_cached(q, cache, table, lengths, dim ** -0.5, *steps(BF16))
    out = ops.attention_cached(q.cuda(), tuple(t.cuda() for t in cache), table.cuda(), ints(lengths))
    within(out, want, bound, "uneven blocks")
    # nothing but zeros
    v_codes.zero_()
    v_scales.fill_(2.0 ** -100)
    assert not ops.attention_cached(q.cuda(), tuple(t.cuda() for t in cache), table.cuda(), ints(lengths)).any()


def test_cached_not_finite(ops) -> None:
    """A NaN scale of a block that a row sees makes the row NaN; beyond the length, or in another head, it does not."""
    lengths, tokens = [40, 40], 16
    table, total = table_for(lengths, tokens, 3)
    for which in (2, 3):
        for dtype in (BF16, F32):
            cache = filled_cache(total, 2, 64, tokens, 4)
            cache[which][table[0, 1].long(), 1] = NAN
            q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(5)).to(dtype)
            out = ops.attention_cached(q.cuda(), tuple(t.cuda() for t in cache), table.cuda(), ints(lengths))
            assert torch.equal(out.isnan().all(2).cpu(), torch.tensor([[0, 0, 1, 1], [0, 0, 0, 0]]).bool())
            assert torch.equal(out.isnan().any(2).cpu(), out.isnan().all(2).cpu())
            shorter = ops.attention_cached(q.cuda(), tuple(t.cuda() for t in cache), table.cuda(), ints([16, 40]))
            assert torch.isfinite(shorter).all()
    cache = filled_cache(total, 2, 64, tokens, 4)
    for bad in (NAN, INF):
        q = torch.ones(2, 4, 64, dtype=BF16)
        q[1, 2, 7] = bad
        out = ops.attention_cached(q.cuda(), tuple(t.cuda() for t in cache), table.cuda(), ints(lengths))
        assert torch.equal(out.isnan().all(2).cpu(), torch.tensor([[0, 0, 0, 0], [0, 0, 1, 0]]).bool())


def test_cached_strided_queries(ops) -> None:
    lengths = [70, 133]
    table, total = table_for(lengths, 32, 1)
    cache = filled_cache(total, 2, 64, 32, 2)
    moved = tuple(t.cuda() for t in cache)
    fused = torch.randn(2, 3, 8 * 64 + 1, generator=torch.Generator().manual_seed(3)).to(BF16)
    for q in (fused[..., :4 * 64].unflatten(2, (4, 64)), fused[..., 1:4 * 64 + 1].unflatten(2, (4, 64)),
              fused[..., :4 * 64].unflatten(2, (64, 4)).transpose(2, 3)):
        want, bound = ref.attention_cached(q, cache, table, lengths, 0.125, *steps(BF16))
        q_dev = torch.empty_strided(q.shape, q.stride(), dtype=BF16, device="cuda").copy_(q)
        within(ops.attention_cached(q_dev, moved, table.cuda(), ints(lengths)), want, bound, "strided q")
    wide = torch.full((2, table.shape[1] + 3), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    q = fused[:, 0, :256].unflatten(1, (4, 64))
    a = ops.attention_cached(q.cuda(), moved, wide.cuda()[:, :table.shape[1]], ints(lengths))
    assert torch.equal(a, ops.attention_cached(q.cuda(), moved, table.cuda(), ints(lengths)))


def test_bad_blocks_raise_a_status_bit(ops) -> None:
    from helion_mlir_backend import native

    lengths = [40, 40]
    good, total = table_for(lengths, 16, 3)
    cache = tuple(t.cuda() for t in filled_cache(total, 1, 64, 16, 4))
    before = host_copy(tuple(t.cpu() for t in cache))
    q = torch.ones(2, 2, 64, dtype=BF16, device="cuda")
    for entry in (-1, total, 2 ** 31 - 1, -2 ** 31):
        table = good.clone()
        table[0, 1] = entry
        out = ops.attention_cached(q, cache, table.cuda(), ints(lengths))
        assert native.kernel_status() == 512
        assert out[0].isnan().all() and torch.isfinite(out[1]).all()
        k, v = ops.cache_read(cache, table.cuda(), ints([0, 0]), ints(lengths), ints([0, 40, 80]), 80, F32)
        assert native.kernel_status() == 512
        for t in (k, v):
            assert t[16:32].isnan().all() and torch.isfinite(t[:16]).all() and torch.isfinite(t[32:]).all()
        x = torch.ones(1, 1, 64, dtype=BF16, device="cuda")
        ops.cache_append(cache, x, x, table[:1].cuda(), ints([17]))
        assert native.kernel_status() == 512
        for now, then in zip(cache, before):
            assert torch.equal(now.cpu(), then)
    # lengths beyond the table
    out = ops.attention_cached(q, cache, good.cuda(), ints([40, 4000]))
    assert native.kernel_status() == 512 and out[1].isnan().all() and torch.isfinite(out[0]).all()
    ops.cache_append(cache, q[:, :1], q[:, :1], good.cuda(), ints([48, 2 ** 31 - 1]))
    assert native.kernel_status() == 512
    for now, then in zip(cache, before):
        assert torch.equal(now.cpu(), then)
    # negative lengths hold nothing
    assert not ops.attention_cached(q, cache, good.cuda(), ints([-5, -2 ** 31])).any()


def test_prompt_then_tokens(ops) -> None:
    """A serving run: prompts through packed attention and into the cache, a second chunk over the prefix read back,
    then single tokens; and the whole again from a captured graph that replays with growing lengths."""
    heads, kv_heads, dim, tokens, prompts = 4, 2, 64, 16, [37, 5, 64]
    gen = torch.Generator().manual_seed(1)
    steps_after, chunk = 20, [9, 30, 1]
    total = [p + c + steps_after for p, c in zip(prompts, chunk)]
    table, blocks = table_for(total, tokens, 2)
    cache = ops.quantized_cache(blocks, kv_heads, dim, tokens)
    host = tuple(t.cpu().clone() for t in cache)
    table_dev = table.cuda()

    def tokens_of(rows):
        return [torch.randn(rows, h, dim, generator=gen).to(BF16) for h in (heads, kv_heads, kv_heads)]

    def on_host(k, v, lengths, at):
        ref.append(host[0], host[2], k, table, lengths, at)
        ref.append(host[1].transpose(2, 3), host[3], v, table, lengths, at)

    at = offsets_of(prompts)
    q, k, v = tokens_of(at[-1])
    want, bound = ref.attention_packed(q, k, v, at, at, dim ** -0.5, True, p_step(BF16))
    within(ops.attention_packed(q.cuda(), k.cuda(), v.cuda(), ints(at)), want, bound, "prompt")
    ops.cache_append(cache, k.cuda(), v.cuda(), table_dev, ints([0, 0, 0]), ints(at))
    on_host(k, v, [0, 0, 0], at)
    # a second chunk: appended, the whole read back, attended to
    lengths = [p + c for p, c in zip(prompts, chunk)]
    at, k_at = offsets_of(chunk), offsets_of(lengths)
    q, k, v = tokens_of(at[-1])
    ops.cache_append(cache, k.cuda(), v.cuda(), table_dev, ints(prompts), ints(at))
    on_host(k, v, prompts, at)
    got = ops.cache_read(cache, table_dev, ints([0, 0, 0]), ints(lengths), ints(k_at), k_at[-1])
    want, bound = ref.attention_packed(q, got[0].cpu(), got[1].cpu(), at, k_at, dim ** -0.5, True, p_step(BF16))
    within(ops.attention_packed(q.cuda(), *got, ints(at), ints(k_at)), want, bound, "second chunk")
    # single tokens, eager and replayed
    q_dev, k_dev, v_dev = (torch.zeros(3, h, dim, dtype=BF16, device="cuda") for h in (heads, kv_heads, kv_heads))
    held, seen = ints(lengths), ints([n + 1 for n in lengths])

    def step():
        ops.cache_append(cache, k_dev, v_dev, table_dev, held)
        return ops.attention_cached(q_dev, cache, table_dev, seen)

    graph, out = None, None
    for i in range(steps_after):
        q, k, v = tokens_of(3)
        q_dev.copy_(q), k_dev.copy_(k), v_dev.copy_(v)
        if i < 3:
            out = step()
        else:
            if graph is None:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    out = step()
            graph.replay()
        on_host(k, v, lengths, [0, 1, 2, 3])
        lengths = [n + 1 for n in lengths]
        want, bound = ref.attention_cached(q[:, None], host, table, lengths, dim ** -0.5, *steps(BF16))
        within(out[:, None], want, bound, f"token {i}")
        held += 1
        seen += 1
    for now, then in zip(cache, host):
        assert torch.equal(now.cpu(), then)


def test_two_streams_at_once(ops) -> None:
    """Calls on two streams, each with its own operands and workspace, answer as they do one after the other."""
    lengths = [700, 90]
    table, total = table_for(lengths, 16, 3)
    cache = tuple(t.cuda() for t in filled_cache(total, 2, 128, 16, 4))
    table_dev, lengths_dev = table.cuda(), ints(lengths)
    queries = [torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(i)).to(BF16).cuda() for i in range(2)]
    want = [ops.attention_cached(q, cache, table_dev, lengths_dev) for q in queries]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.attention_cached(queries[i], cache, table_dev, lengths_dev))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
