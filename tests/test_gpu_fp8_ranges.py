"""Attention over the 8-bit KV cache where its running maxima, sums and merges are stretched (GPU).

Compared with 64-bit attention over the values the cache holds, within the bounds that
``fp8_reference.attention`` derives.
"""

from __future__ import annotations

import pytest
import torch

from tests.fp8_reference import attention, make_cache, rows_of, tables_for
from tests.test_gpu_fp8_attention import check_decode, check_prefill, decode, prefill
from tokenserve_b200 import ops

pytestmark = pytest.mark.gpu

BF, FH = torch.bfloat16, torch.float16


@pytest.mark.parametrize(("hq", "hkv", "d"), [(8, 1, 128), (16, 1, 128), (7, 1, 64)])
def test_merges_of_many_partials_are_the_same_on_every_launch(cuda_device, hq, hkv, d) -> None:  # type: ignore[no-untyped-def]
    """A long sequence's partials are merged by groups, each group into its first partial's place,
    which every lane of the merging warp has read by then."""
    gen = torch.Generator(device=cuda_device).manual_seed(hq)
    lens = [16000, 40, 5000, 700]
    nb, tab = tables_for(lens, 16, gen)
    cache = make_cache(gen, nb, hkv, 16, d)
    q = torch.randn(len(lens), hq, d, generator=gen, device=cuda_device).to(BF)
    ctx = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    first = decode(q, cache, tab, ctx)
    check_decode(first, q, cache, tab, lens)
    for _ in range(30):
        assert torch.equal(decode(q, cache, tab, ctx), first)


@pytest.mark.parametrize(("dtype", "hq", "hkv", "d"), [(BF, 8, 8, 128), (FH, 4, 1, 64), (BF, 16, 1, 128)])
def test_chunks_whose_last_key_tiles_some_warps_do_not_see(cuda_device, dtype, hq, hkv, d) -> None:  # type: ignore[no-untyped-def]
    """A warp's 32 rows end before a tile of keys that later rows of its query tile see."""
    gen = torch.Generator(device=cuda_device).manual_seed(hq + d)
    chunks, ctxs = [128, 97, 256, 64], [128, 161, 300, 65]
    nb, tab = tables_for(ctxs, 16, gen)
    cache = make_cache(gen, nb, hkv, 16, d)
    q = torch.randn(sum(chunks), hq, d, generator=gen, device=cuda_device).to(dtype)
    qsl = torch.tensor([0, *chunks], device=cuda_device).cumsum(0).to(torch.int32)
    ctx = torch.tensor(ctxs, dtype=torch.int32, device=cuda_device)
    first = prefill(q, cache, tab, qsl, ctx, max(chunks))
    check_prefill(first, q, cache, tab, chunks, ctxs)
    for _ in range(10):
        assert torch.equal(prefill(q, cache, tab, qsl, ctx, max(chunks)), first)


def zero_rows(cache, tab, i, rows, keys=True):  # type: ignore[no-untyped-def]
    """Positions ``rows`` of sequence i hold what an all-zero V (and K) row is stored as."""
    kp, vp, ks, vs = cache
    for pool, sc in ((vp, vs), (kp, ks)) if keys else ((vp, vs),):
        for p in rows:
            blk = int(tab[i, p // 16])
            pool.view(torch.uint8)[blk, :, p % 16] = 0
            sc[blk, :, p % 16] = 2.0**-126


ZERO_LENS = [4, 36, 70, 100, 400, 1300, 1300, 5000, 9000]
ZERO_ROWS = [range(3), range(32), range(64), range(64), range(32, 300), range(1000), range(300, 1299),
             range(2500), range(4, 9000)]  # fmt: skip


@pytest.mark.parametrize("magnitude", [2.0**-60, 2.0**-7, 1.0, 2.0**20, 2.0**60])
@pytest.mark.parametrize(("hq", "hkv", "equal"), [(8, 1, True), (8, 1, False), (32, 8, False), (16, 1, True)])
def test_decode_with_runs_of_zero_value_rows(cuda_device, magnitude, hq, hkv, equal) -> None:  # type: ignore[no-untyped-def]
    """Zero rows at the start, in the middle and to the end of a context, within one partition and
    over many: each counts in the softmax's sum and adds nothing to the output."""
    gen = torch.Generator(device=cuda_device).manual_seed(21)
    nb, tab = tables_for(ZERO_LENS, 16, gen)
    cache = make_cache(gen, nb, hkv, 16, 128)
    if equal:
        cache[2].zero_()
    else:
        cache[2].mul_(8)
    cache[3].mul_(magnitude)
    for i, rows in enumerate(ZERO_ROWS):
        zero_rows(cache, tab, i, rows, keys=equal or i % 2 == 0)
    q = torch.randn(len(ZERO_LENS), hq, 128, generator=gen, device=cuda_device).to(BF)
    ctx = torch.tensor(ZERO_LENS, dtype=torch.int32, device=cuda_device)
    check_decode(decode(q, cache, tab, ctx), q, cache, tab, ZERO_LENS)


def test_decode_after_a_prompt_of_zero_rows_through_the_append(cuda_device) -> None:  # type: ignore[no-untyped-def]
    """64 zero rows, then ordinary ones, written by the operator itself; scores of spread 1."""
    gen = torch.Generator(device=cuda_device).manual_seed(22)
    n, zeros = 130, 64
    nb, tab = tables_for([n], 16, gen)
    kp = torch.zeros(nb, 1, 16, 128, dtype=torch.uint8, device=cuda_device).view(torch.float8_e4m3fn)
    vp, ks = kp.clone(), torch.zeros(nb, 1, 16, device=cuda_device)
    cache = (kp, vp, ks, ks.clone())
    k, v = (torch.randn(n, 1, 128, generator=gen, device=cuda_device).to(BF) for _ in range(2))
    v[:zeros] = 0
    pos = torch.arange(n, device=cuda_device)
    slots = tab[0, pos // 16].long() * 16 + pos % 16
    ops.reshape_and_cache_fp8(k, v, *cache, slots)
    q = torch.randn(1, 4, 128, generator=gen, device=cuda_device).to(BF)
    ctx = torch.tensor([n], dtype=torch.int32, device=cuda_device)
    check_decode(decode(q, cache, tab, ctx), q, cache, tab, [n])


@pytest.mark.parametrize("span", [20, 40, 60])
def test_decode_of_value_rows_over_many_binades(cuda_device, span) -> None:  # type: ignore[no-untyped-def]
    """Whole blocks, and single rows, of very large and very small values."""
    gen = torch.Generator(device=cuda_device).manual_seed(span)
    lens = [40, 333, 2500, 7000]
    nb, tab = tables_for(lens, 16, gen)
    kp, vp, ks, vs = make_cache(gen, nb, 2, 16, 128)
    wide = lambda *s: torch.exp2(torch.randint(-span, span + 1, s, generator=gen,  # noqa: E731
                                               device=cuda_device).float())  # fmt: skip
    vs[::2] *= wide(len(vs[::2]), 1, 1)
    vs[1::2] *= wide(*vs[1::2].shape)
    q = torch.randn(len(lens), 8, 128, generator=gen, device=cuda_device).to(BF)
    ctx = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    check_decode(decode(q, (kp, vp, ks, vs), tab, ctx), q, (kp, vp, ks, vs), tab, lens)


def check_prefill_wide(out, q, cache, tab, chunks, ctxs):  # type: ignore[no-untyped-def]
    at = 0
    for i, (n, c) in enumerate(zip(chunks, ctxs, strict=True)):
        rows = slice(at, at + n)
        at += n
        want, off = attention(q[rows], *rows_of(cache[0], cache[2], tab[i], c),
                              *rows_of(cache[1], cache[3], tab[i], c), q.shape[-1] ** -0.5, c - n)
        got, most = out[rows].double(), torch.finfo(q.dtype).max
        # An output past the type's largest number is that type's infinity (fp16: past 65504).
        past = (want.abs() + off > most) & torch.isinf(got) & (got * want > 0)
        bad = ((got - want).abs() - off).masked_fill(past, 0.0)
        assert (bad <= 0).all(), (i, n, c, float(bad.max()))


WIDE_CHUNKS, WIDE_CTX = [40, 150, 64, 1], [900, 150, 64, 700]


@pytest.mark.parametrize(("dtype", "hq", "hkv", "d"), [(BF, 8, 2, 128), (FH, 8, 2, 128), (FH, 4, 4, 64)])
@pytest.mark.parametrize("kind", ["blocks", "rows", "outlier", "growing", "zeros"])
def test_prefill_of_value_rows_over_many_binades(cuda_device, dtype, hq, hkv, d, kind) -> None:  # type: ignore[no-untyped-def]
    """Within the bound for exact K and V codes: blocks of 32 tokens and single rows of magnitudes 2^+-20, a row 2^24 times larger than all
    others whose softmax weight is nothing, magnitudes that grow along the context, runs of zeros."""
    gen = torch.Generator(device=cuda_device).manual_seed(31)
    nb, tab = tables_for(WIDE_CTX, 16, gen)
    cache = make_cache(gen, nb, hkv, 16, d)
    kp, vp, ks, vs = cache
    q = torch.randn(sum(WIDE_CHUNKS), hq, d, generator=gen, device=cuda_device).abs().to(dtype)
    wide = lambda *s: torch.exp2(torch.randint(-20, 21, s, generator=gen,  # noqa: E731
                                               device=cuda_device).float())  # fmt: skip
    for i, c in enumerate(WIDE_CTX):
        blocks = tab[i, : -(-c // 16)].long()
        if kind == "blocks":
            vs[blocks] *= wide(len(blocks) // 2 + 1, 1, 1).repeat_interleave(2, 0)[: len(blocks)]
        elif kind == "rows":
            vs[blocks] *= wide(*vs[blocks].shape)
        elif kind == "growing":
            vs[blocks] *= torch.exp2(torch.arange(len(blocks), device=cuda_device) - 20.0)[:, None, None]
        elif kind == "zeros":
            zero_rows(cache, tab, i, [range(0), range(96), range(20, 40), range(650)][i], keys=i == 1)
        else:  # codes of K all negative, q positive: a score of about -100
            blk = blocks[len(blocks) // 3]
            kp.view(torch.uint8)[blk, :, 5] = 0xF0
            ks[blk, :, 5] = 0.03
            vs[blk, :, 5] *= 2.0**24
    qsl = torch.tensor([0, *WIDE_CHUNKS], device=cuda_device).cumsum(0).to(torch.int32)
    ctx = torch.tensor(WIDE_CTX, dtype=torch.int32, device=cuda_device)
    out = prefill(q, cache, tab, qsl, ctx, max(WIDE_CHUNKS))
    check_prefill_wide(out, q, cache, tab, WIDE_CHUNKS, WIDE_CTX)


@pytest.mark.parametrize("which", ["key", "value"])
@pytest.mark.parametrize(("hq", "hkv", "d"), [(8, 1, 128), (16, 1, 64)])
def test_decode_of_a_nan_row_wherever_it_stands(cuda_device, which, hq, hkv, d) -> None:  # type: ignore[no-untyped-def]
    """The only token, the only one of a last block or of a last partition, all tokens of a context,
    one in the middle of many partitions: the sequence's rows become NaN, the others stay clean."""
    gen = torch.Generator(device=cuda_device).manual_seed(41)
    lens = [1, 17, 65, 129, 400, 2049, 9000, 50]
    bad = [range(1), range(16, 17), range(64, 65), range(129), range(399, 400), range(2048, 2049),
           range(4444, 4445), range(0)]  # fmt: skip
    nb, tab = tables_for(lens, 16, gen)
    cache = make_cache(gen, nb, hkv, 16, d)
    for i, rows in enumerate(bad):
        for p in rows:
            for pool, sc in (((cache[0], cache[2]) if which == "key" else (cache[1], cache[3])),):
                pool.view(torch.uint8)[int(tab[i, p // 16]), :, p % 16] = 0x7F
                sc[int(tab[i, p // 16]), :, p % 16] = float("nan")
    q = torch.randn(len(lens), hq, d, generator=gen, device=cuda_device).to(BF)
    ctx = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    out = decode(q, cache, tab, ctx)
    assert torch.isnan(out[:-1]).all()
    check_decode(out[-1:], q[-1:], cache, tab[-1:], lens[-1:])
    qsl = torch.arange(len(lens) + 1, dtype=torch.int32, device=cuda_device)
    out = prefill(q, cache, tab, qsl, ctx, 1)
    assert torch.isnan(out[:-1]).all()
    check_prefill(out[-1:], q[-1:], cache, tab[-1:], [1], lens[-1:])


def exact(q, cache, tab, chunks, ctxs):  # type: ignore[no-untyped-def]
    """The attention in 64 bits, ``[T, Hq, D]``."""
    out, at = [], 0
    for i, (n, c) in enumerate(zip(chunks, ctxs, strict=True)):
        out.append(attention(q[at : at + n], *rows_of(cache[0], cache[2], tab[i], c),
                             *rows_of(cache[1], cache[3], tab[i], c), q.shape[-1] ** -0.5, c - n)[0])  # fmt: skip
        at += n
    return torch.cat(out)


@pytest.mark.parametrize(("hq", "hkv", "d"), [(8, 2, 128), (4, 4, 64), (16, 1, 128)])
def test_fp16_outputs_lose_little_beside_their_own_rounding(cuda_device, hq, hkv, d) -> None:  # type: ignore[no-untyped-def]
    """Codes are exact in the tiles, so what is left beside the output's rounding is one rounding of
    the weights, to 11 bits as well: two independent errors of one size in the 2-norm, sqrt(2) times
    the output's rounding together (a row's weights average theirs, so less than that of each row)."""
    gen = torch.Generator(device=cuda_device).manual_seed(51)
    chunks, ctxs = [200, 64, 1, 300], [700, 64, 900, 300]
    nb, tab = tables_for(ctxs, 16, gen)
    cache = make_cache(gen, nb, hkv, 16, d)
    q = torch.randn(sum(chunks), hq, d, generator=gen, device=cuda_device).to(FH)
    qsl = torch.tensor([0, *chunks], device=cuda_device).cumsum(0).to(torch.int32)
    ctx = torch.tensor(ctxs, dtype=torch.int32, device=cuda_device)
    want = exact(q, cache, tab, chunks, ctxs)
    own = (want.to(FH).double() - want).norm()
    got = prefill(q, cache, tab, qsl, ctx, max(chunks)).double()
    assert (got - want).norm() <= 1.5 * own, float((got - want).norm() / own)
    check_prefill(got.to(FH), q, cache, tab, chunks, ctxs, k_half=0.0)


@pytest.mark.parametrize(("dtype", "d"), [(BF, 128), (FH, 64)])
def test_zero_rows_that_take_nearly_all_weight(cuda_device, dtype, d) -> None:  # type: ignore[no-untyped-def]
    """Positions 20..39 hold zero V rows with scores about 2^70 times the others' weights, so the
    outputs (bf16: 2^-70 of V) come from the small weights of the other rows alone."""
    gen = torch.Generator(device=cuda_device).manual_seed(61)
    chunks, ctxs = [60, 5], [90, 200]
    nb, tab = tables_for(ctxs, 16, gen)
    cache = make_cache(gen, nb, 2, 16, d)
    kp, vp, ks, vs = cache
    if dtype == FH:  # outputs of fp16's normal range
        vs.mul_(2.0**60)
    q = torch.randn(sum(chunks), 8, d, generator=gen, device=cuda_device).abs().to(dtype)
    want = 48.0 / (0.8 * d**0.5)  # K's value that gives q's mean row a score of 48 (2^70)
    for i in range(2):
        zero_rows(cache, tab, i, range(20, 40), keys=False)
        for p in range(20, 40):
            kp.view(torch.uint8)[int(tab[i, p // 16]), :, p % 16] = 0x70  # 128
            ks[int(tab[i, p // 16]), :, p % 16] = want / 128
    qsl = torch.tensor([0, *chunks], device=cuda_device).cumsum(0).to(torch.int32)
    ctx = torch.tensor(ctxs, dtype=torch.int32, device=cuda_device)
    out = prefill(q, cache, tab, qsl, ctx, max(chunks))
    check_prefill_wide(out, q, cache, tab, chunks, ctxs)
    check_decode(decode(q[59:61], cache, tab, ctx), q[59:61], cache, tab, ctxs)


@pytest.mark.parametrize("scale", [-0.11, 0.0, 3.0])
@pytest.mark.parametrize(("dtype", "hq", "hkv", "d"), [(BF, 8, 2, 128), (FH, 12, 1, 64), (torch.float32, 4, 2, 64)])
def test_softmax_scales_of_any_sign(cuda_device, scale, dtype, hq, hkv, d) -> None:  # type: ignore[no-untyped-def]
    gen = torch.Generator(device=cuda_device).manual_seed(71)
    chunks, ctxs = [70, 5], [200, 333]
    nb, tab = tables_for(ctxs, 16, gen)
    cache = make_cache(gen, nb, hkv, 16, d)
    q = torch.randn(sum(chunks), hq, d, generator=gen, device=cuda_device).to(dtype)
    qsl = torch.tensor([0, *chunks], device=cuda_device).cumsum(0).to(torch.int32)
    ctx = torch.tensor(ctxs, dtype=torch.int32, device=cuda_device)
    n = ops.decode_workspace_size(2, hq, hkv, d, tab.shape[1], 16, dtype)
    ws = torch.empty(max(n, 256), dtype=torch.uint8, device=cuda_device)
    pre, dec, at = torch.full_like(q, 7.0), torch.full_like(q[:2], 7.0), 0
    ops.paged_prefill_fp8(pre, q, *cache, tab, qsl, ctx, max(chunks), scale)
    ops.paged_decode_fp8(dec, q[:2], *cache, tab, ctx, scale, ws)
    for i, (n, c) in enumerate(zip(chunks, ctxs, strict=True)):
        rows = (*rows_of(cache[0], cache[2], tab[i], c), *rows_of(cache[1], cache[3], tab[i], c))
        for got, x, pos in ((pre[at : at + n], q[at : at + n], c - n), (dec[i : i + 1], q[i : i + 1], None)):
            want, off = attention(x, *rows, scale, pos)
            assert ((got.double() - want).abs() <= off).all()
        at += n


@pytest.mark.parametrize(("hq", "hkv", "d"), [(32, 1, 128), (100, 1, 64), (128, 1, 128), (66, 2, 128)])
def test_prefill_of_many_query_heads_per_kv_head(cuda_device, hq, hkv, d) -> None:  # type: ignore[no-untyped-def]
    """Up to 128 rows of a tile are one token's heads; some of a tile's rows belong to no query."""
    gen = torch.Generator(device=cuda_device).manual_seed(hq)
    chunks, ctxs = [9, 1, 30], [100, 1, 30]
    nb, tab = tables_for(ctxs, 16, gen)
    cache = make_cache(gen, nb, hkv, 16, d)
    q = torch.randn(sum(chunks), hq, d, generator=gen, device=cuda_device).to(BF)
    qsl = torch.tensor([0, *chunks], device=cuda_device).cumsum(0).to(torch.int32)
    ctx = torch.tensor(ctxs, dtype=torch.int32, device=cuda_device)
    check_prefill(prefill(q, cache, tab, qsl, ctx, max(chunks)), q, cache, tab, chunks, ctxs, k_half=0.0)
