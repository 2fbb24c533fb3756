"""Attention over the 8-bit KV cache where its running maxima, sums and merges are stretched (GPU).

Compared with 64-bit attention over the values the cache holds, within the bounds that
``fp8_reference.attention`` derives.
"""

from __future__ import annotations

import pytest
import torch

from tests.fp8_reference import make_cache, tables_for
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
