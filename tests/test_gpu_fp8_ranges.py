"""Attention over the 8-bit KV cache where its running maxima, sums and merges are stretched (GPU).

Compared with 64-bit attention over the values the cache holds, within the bounds that
``fp8_reference.attention`` derives.
"""

from __future__ import annotations

import pytest
import torch

from tests.fp8_reference import make_cache, tables_for
from tests.test_gpu_fp8_attention import check_decode, check_prefill, decode, prefill

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
