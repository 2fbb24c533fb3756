"""Codes and scales of the 8-bit KV cache, bit for bit as the format states them (GPU).

scale = max(amax / 448, 2^-126) and code = e4m3(x / scale), the quotients in float32 rounded to
nearest even and then to e4m3: torch's division of tensors and its conversion do the same (a
division by a Python number multiplies by its reciprocal instead). Signs of zeros apart.
"""

from __future__ import annotations

import pytest
import torch

from tests.fp8_reference import E4M3
from tokenserve_b200 import ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def append(rows, d, h=1, odd=False):  # type: ignore[no-untyped-def]
    """Codes and scales of rows ``[T, h, d]`` written at slots 0.."""
    t, dev = rows.shape[0], rows.device
    if odd:  # one element past a 16-byte boundary: the scalar kernel
        buf = torch.zeros(t, h * d + 1, dtype=rows.dtype, device=dev)
        buf[:, 1:] = rows.flatten(1)
        rows = buf[:, 1:].unflatten(1, (h, d))
    nb = -(-t // 16)
    kp = torch.zeros(nb, h, 16, d, dtype=torch.uint8, device=dev).view(E4M3)
    vp, ks = kp.clone(), torch.zeros(nb, h, 16, device=dev)
    vs = ks.clone()
    ops.reshape_and_cache_fp8(rows, rows, kp, vp, ks, vs, torch.arange(t, device=dev))
    flat = lambda x: x.transpose(1, 2).flatten(0, 1)[:t]  # noqa: E731
    assert torch.equal(kp.view(torch.uint8), vp.view(torch.uint8)) and torch.equal(ks, vs)
    return flat(kp.view(torch.uint8)).view(E4M3), flat(ks)


def check(rows, code, scale):  # type: ignore[no-untyped-def]
    x = rows.float()
    want = (x.abs().amax(-1) / torch.full_like(x[..., 0], 448)).clamp_min(2.0**-126)
    assert torch.equal(scale, want)
    q = (x / want[..., None]).clamp(-448, 448).to(E4M3)
    assert (code.float() == q.float()).all(), int((code.float() != q.float()).sum())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("d", "odd"), [(64, False), (128, False), (256, False), (128, True), (80, False)])
def test_codes_are_the_rounded_quotients(cuda_device, dtype, d, odd) -> None:  # type: ignore[no-untyped-def]
    gen = torch.Generator(device=cuda_device).manual_seed(d)
    rows = torch.randn(60000, 2, d, generator=gen, device=cuda_device)
    rows = (rows * torch.exp(torch.randn(60000, 2, 1, generator=gen, device=cuda_device))).to(dtype)
    check(rows, *append(rows, d, 2, odd))


@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("binade", [-140, -126, -118, -110, -90, -60, -14, 0, 9, 100, 127])
def test_codes_of_values_at_the_middles(cuda_device, binade, odd) -> None:  # type: ignore[no-untyped-def]
    """Values at, and float32 steps around, the middles between codes, for rows of any magnitude."""
    gen = torch.Generator(device=cuda_device).manual_seed(binade + 200)
    codes = torch.arange(0, 127, dtype=torch.uint8, device=cuda_device).view(E4M3).double()
    mid = (codes[:-1] + codes[1:]) / 2
    t, d = 2000, 128
    amax = (1 + torch.rand(t, 1, generator=gen, device=cuda_device)) * 2.0**min(binade, 126)
    scale = (amax / torch.full_like(amax, 448)).clamp_min(2.0**-126).double()
    pick = mid[torch.randint(0, len(mid), (t, d), generator=gen, device=cuda_device)]
    step = torch.randint(-3, 4, (t, d), generator=gen, device=cuda_device).double()
    x = (pick * scale * (1 + step * 2.0**-24)).float()
    x = torch.minimum(x, amax) * (1 - 2 * torch.randint(0, 2, (t, d), generator=gen, device=cuda_device))
    x[:, 7:8] = amax
    check(x[:, None], *append(x[:, None], d, 1, odd))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("d", "rd"), [(64, 64), (128, 64), (80, 20)])
def test_both_writing_operators_give_the_same_codes(cuda_device, dtype, d, rd) -> None:  # type: ignore[no-untyped-def]
    """K at angle 0 and V of the fused projection, through rotary_and_cache."""
    gen = torch.Generator(device=cuda_device).manual_seed(rd)
    t, hq, hkv = 1500, 3, 2
    qkv = torch.randn(t, hq + 2 * hkv, d, generator=gen, device=cuda_device)
    mag = torch.exp2(torch.randint(-8, 8, (t, 1, 1), generator=gen, device=cuda_device).float())
    mag[0] = 2.0**-100  # a scale too small for its quotients' residuals (fp16: zeros)
    qkv = (qkv * mag).to(dtype)
    nb = -(-t // 16)
    kp = torch.zeros(nb, hkv, 16, d, dtype=torch.uint8, device=cuda_device).view(E4M3)
    vp, ks = kp.clone(), torch.zeros(nb, hkv, 16, device=cuda_device)
    vs = ks.clone()
    q = torch.empty(t, hq, d, dtype=dtype, device=cuda_device)
    at = torch.arange(t, device=cuda_device)
    ops.rotary_and_cache(qkv.flatten(1), q, kp, vp, at, at, torch.zeros(rd // 2, device=cuda_device),
                         hq, hkv, key_scales=ks, value_scales=vs)  # fmt: skip
    flat = lambda x: x.transpose(1, 2).flatten(0, 1)[:t]  # noqa: E731
    for pool, sc, first in ((kp, ks, hq), (vp, vs, hq + hkv)):
        check(qkv[:, first : first + hkv], flat(pool.view(torch.uint8)).view(E4M3), flat(sc))
    assert torch.equal(q, qkv[:, :hq])
