"""Attention over the 8-bit KV cache where its running maxima, sums and merges are stretched (GPU).

Compared with 64-bit attention over the values the cache holds, within the bounds that
``fp8_reference.attention`` derives.
"""

from __future__ import annotations

import pytest
import torch

from tests.fp8_reference import make_cache, tables_for
from tests.test_gpu_fp8_attention import check_decode, decode

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
