"""Writing the 8-bit KV cache, rotary positions fused with the write, and reading back (GPU).

References are computed in 64 bits. Tolerances: a code is at most half an e4m3 step from
x / scale (2^-4 of it, 2^-10 among the subnormals), times 1 + 2^-21 for the fp32 reciprocal and
product; a scale is within 2^-23 of amax / 448. A rotary value is a sum of two products whose cos
and sin are off by at most 2^-21 (the fraction of a turn rounded to fp32 moves the angle by
2 pi 2^-26, sincospif and the factor's product add 2^-23), with three fp32 roundings: together
under 2^-20 (|a| + |b|) times the factor, then half a step of the output type.
"""

from __future__ import annotations

import pytest
import torch

from tests.fp8_reference import E4M3, HALF_STEP, make_cache, rounded, rows_of, tables_for
from tokenserve_b200 import ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def empty_cache(nb, h, bs, d, dev):  # type: ignore[no-untyped-def]
    """Pools filled with a pattern no write produces, so untouched slots can be told."""
    kp = torch.full((nb, h, bs, d), 0x55, dtype=torch.uint8, device=dev).view(E4M3)
    ks = torch.full((nb, h, bs), 123.0, device=dev)
    return kp, kp.clone(), ks, ks.clone()


def slots_for(n, nb, bs, gen, pad=0):  # type: ignore[no-untyped-def]
    s = torch.randperm(nb * bs, generator=gen, device=gen.device)[:n].long()
    if pad:
        s[::pad] = -1
    return s


def check_rows(x, pool, scales, slots, bs, slack=0.0, near=None):  # type: ignore[no-untyped-def]
    """Rows ``x [T, H, D]`` (64 bits) against codes and scales at their slots. ``near [T, H, D]``:
    how far the kernel's own fp32 rows may be from x before they are quantised."""
    live = slots >= 0
    x, blk, off = x[live], slots[live] // bs, slots[live] % bs
    code = pool.view(torch.uint8)[blk, :, off].view(E4M3).double()
    sc = scales[blk, :, off].double()
    near = torch.zeros_like(x) if near is None else near[live]
    want = (x.abs().amax(-1) / 448).clamp_min(2.0**-126)
    assert ((sc - want).abs() <= want * 2.0**-23 + near.amax(-1) / 448).all()
    y = x / sc[..., None]
    half = (y.abs() * 2.0**-4).clamp_min(2.0**-10) * (1 + 2.0**-21) + 2 * near / sc[..., None]
    assert ((code - y).abs() <= half).all(), float(((code - y).abs() - half).max())
    untouched = torch.ones(pool.shape[0] * bs, dtype=torch.bool, device=pool.device)
    untouched[slots[live]] = False
    u = pool.view(torch.uint8).transpose(1, 2).flatten(0, 1)[untouched]
    assert (u == 0x55).all() and (scales.transpose(1, 2).flatten(0, 1)[untouched] == 123.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(
    ("t", "h", "d", "bs"),
    [(1, 1, 128, 16), (1, 8, 64, 16), (37, 8, 128, 16), (300, 2, 64, 16), (65, 3, 256, 16),
     (33, 2, 32, 8), (19, 2, 80, 16), (9, 1, 7, 5), (1030, 8, 128, 16)],
)  # fmt: skip
@pytest.mark.parametrize("layout", ["whole", "strided", "odd"])
def test_append_quantises_each_row(cuda_device, dtype, t, h, d, bs, layout) -> None:  # type: ignore[no-untyped-def]
    gen = torch.Generator(device=cuda_device).manual_seed(t * 7 + d)
    x = torch.randn(t, 2 * h, d, generator=gen, device=cuda_device)
    x = (x * torch.exp(2 * torch.randn(t, 2 * h, 1, generator=gen, device=cuda_device))).to(dtype)
    if layout == "whole":
        k, v = x[:, :h].contiguous(), x[:, h:].contiguous()
    elif layout == "strided":
        k, v = x[:, :h], x[:, h:]
    else:  # one element past a 16-byte boundary, odd token stride
        buf = torch.zeros(t, 2 * h * d + 3, dtype=dtype, device=cuda_device)
        buf[:, 1 : 1 + 2 * h * d] = x.flatten(1)
        rows = buf[:, 1 : 1 + 2 * h * d].unflatten(1, (2 * h, d))
        k, v = rows[:, :h], rows[:, h:]
    nb = -(-t // bs) + 2
    kp, vp, ks, vs = empty_cache(nb, h, bs, d, cuda_device)
    slots = slots_for(t, nb, bs, gen, pad=5)
    ops.reshape_and_cache_fp8(k, v, kp, vp, ks, vs, slots)
    check_rows(k.double(), kp, ks, slots, bs)
    check_rows(v.double(), vp, vs, slots, bs)


def test_append_of_rows_at_the_ends_of_the_range(cuda_device) -> None:  # type: ignore[no-untyped-def]
    rows = torch.zeros(8, 1, 64, device=cuda_device)
    rows[1, 0, 5] = float("inf")
    rows[2, 0, 63] = float("nan")
    rows[3, 0, :] = 1e-44  # subnormal
    rows[4, 0, 7] = 3.4e38
    rows[5, 0, 0] = -2.0**-100
    rows[6, 0, 3] = -float("inf")
    rows[7, 0, ::2] = 448.0
    kp, vp, ks, vs = empty_cache(2, 1, 16, 64, cuda_device)
    slots = torch.arange(8, device=cuda_device)
    ops.reshape_and_cache_fp8(rows, -rows, kp, vp, ks, vs, slots)
    k, s = kp[0, 0].float(), ks[0, 0]
    for bad in (1, 2, 6):
        assert torch.isnan(s[bad]) and torch.isnan(k[bad]).all()
    assert s[0] == s[3] == 2.0**-126 and (k[0] == 0).all()
    assert k[4, 7] == 448 and k[5, 0] == -448 and (k[7, ::2] == 448).all() and s[7] == 1
    assert torch.equal(vp[0, 0, 7].float(), -k[7])


def test_append_flags_slots_past_the_pool_and_writes_tags(cuda_device) -> None:  # type: ignore[no-untyped-def]
    x = torch.randn(4, 2, 64, device=cuda_device).half()
    kp, vp, ks, vs = empty_cache(2, 2, 16, 64, cuda_device)
    slots = torch.tensor([3, 32, -1, 31], device=cuda_device)
    flag = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    tags = torch.tensor([11, 12, 13, 14], dtype=torch.int32, device=cuda_device)
    tag_pool = torch.full((32,), -1, dtype=torch.int32, device=cuda_device)
    ops.reshape_and_cache_fp8(x, x, kp, vp, ks, vs, slots, token_tags=tags, tag_pool=tag_pool,
                              error_flag=flag)  # fmt: skip
    assert flag.item() == 1
    assert tag_pool[3] == 11 and tag_pool[31] == 14 and int((tag_pool >= 0).sum()) == 2
    slots[1] = -1
    check_rows(x.double(), kp, ks, slots, 16)


def rotate(x, pos, inv_freq, mscale, interleaved):  # type: ignore[no-untyped-def]
    """``x [T, H, D]`` turned, in 64 bits, and how far fp32 arithmetic may be off."""
    half = inv_freq.numel()
    ang = pos.double()[:, None] * inv_freq.double()[None, :]
    c, s = (ang.cos() * mscale)[:, None], (ang.sin() * mscale)[:, None]
    y, near = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = x[..., first].double(), x[..., second].double()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    near[..., first] = near[..., second] = (a.abs() + b.abs()) * mscale * 2.0**-20
    return y, near


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize(
    ("t", "hq", "hkv", "d", "rd", "bs"),
    [(1, 4, 2, 64, 64, 16), (37, 32, 8, 128, 128, 16), (70, 8, 8, 128, 64, 16),
     (5, 14, 2, 64, 32, 16), (9, 6, 3, 80, 20, 16), (3, 2, 1, 10, 6, 4), (260, 8, 1, 256, 128, 16),
     (11, 5, 1, 128, 40, 16)],
)  # fmt: skip
def test_rotary_turns_q_and_k_and_writes_the_cache(
    cuda_device, dtype, interleaved, quant, t, hq, hkv, d, rd, bs  # type: ignore[no-untyped-def]
) -> None:
    gen = torch.Generator(device=cuda_device).manual_seed(t + d)
    qkv = torch.randn(t, (hq + 2 * hkv) * d, generator=gen, device=cuda_device).to(dtype)
    pos = torch.randint(0, 131072, (t,), generator=gen, device=cuda_device)
    pos[0] = 0
    if t > 3:
        pos[1], pos[2] = 1, 2**24 + 1
    inv = (10000.0 ** (-torch.arange(rd // 2, device=cuda_device).double() / (rd // 2))).float()
    mscale = 1.0 if t % 2 else 1.25
    nb = -(-t // bs) + 2
    slots = slots_for(t, nb, bs, gen, pad=4 if t > 1 else 0)
    q = torch.full((t, hq, d), 7.0, dtype=dtype, device=cuda_device)
    kp, vp, ks, vs = empty_cache(nb, hkv, bs, d, cuda_device)
    if not quant:
        kp = torch.full((nb, hkv, bs, d), 7.0, dtype=dtype, device=cuda_device)
        vp, ks, vs = kp.clone(), None, None
    ops.rotary_and_cache(qkv, q, kp, vp, slots, pos, inv, hq, hkv, key_scales=ks, value_scales=vs,
                         interleaved=interleaved, attention_scaling=mscale)  # fmt: skip
    x = qkv.view(t, hq + 2 * hkv, d)
    y, near = rotate(x[:, : hq + hkv], pos, inv, mscale, interleaved)
    off = (q.double() - y[:, :hq]).abs()
    assert (off <= near[:, :hq] + rounded(y[:, :hq], dtype) * (1 + 2.0**-10)).all()
    if quant:
        check_rows(y[:, hq:], kp, ks, slots, bs, near=near[:, hq:])
        check_rows(x[:, hq + hkv :].double(), vp, vs, slots, bs)
        return
    live = slots >= 0
    blk, o = slots[live] // bs, slots[live] % bs
    off = (kp[blk, :, o].double() - y[live][:, hq:]).abs()
    assert (off <= near[live][:, hq:] + rounded(y[live][:, hq:], dtype) * (1 + 2.0**-10)).all()
    assert torch.equal(vp[blk, :, o], x[live][:, hq + hkv :])
    rest = torch.ones(nb * bs, dtype=torch.bool, device=cuda_device)
    rest[slots[live]] = False
    assert (kp.transpose(1, 2).flatten(0, 1)[rest] == 7).all()


def test_rotary_on_padded_projection_rows(cuda_device) -> None:  # type: ignore[no-untyped-def]
    """A token stride beyond the row, and a base one element past a 16-byte boundary."""
    t, hq, hkv, d = 6, 4, 2, 64
    width = (hq + 2 * hkv) * d
    buf = torch.randn(t, width + 8, device=cuda_device).bfloat16()
    inv = torch.rand(d // 2, device=cuda_device)
    pos = torch.arange(t, device=cuda_device) * 1000
    slots = torch.arange(t, device=cuda_device)
    got = []
    for rows in (buf[:, :width], buf[:, 1 : width + 1], buf[:, 1 : width + 1].contiguous()):
        kp, vp, ks, vs = empty_cache(1, hkv, 16, d, cuda_device)
        q = torch.zeros(t, hq, d, dtype=torch.bfloat16, device=cuda_device)
        ops.rotary_and_cache(rows, q, kp, vp, slots, pos, inv, hq, hkv, key_scales=ks,
                             value_scales=vs)  # fmt: skip
        y, near = rotate(rows.reshape(t, -1, d)[:, : hq + hkv], pos, inv, 1.0, False)
        assert ((q.double() - y[:, :hq]).abs()
                <= near[:, :hq] + rounded(y[:, :hq], q.dtype) * (1 + 2.0**-10)).all()  # fmt: skip
        check_rows(y[:, hq:], kp, ks, slots, 16, near=near[:, hq:])
        got.append((q, kp.view(torch.uint8)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(
    ("h", "d", "bs"), [(8, 128, 16), (2, 64, 16), (1, 256, 8), (3, 80, 16), (1, 9, 3)]
)
def test_read_back_gives_code_times_scale(cuda_device, dtype, h, d, bs) -> None:  # type: ignore[no-untyped-def]
    gen = torch.Generator(device=cuda_device).manual_seed(d)
    lens = [0, 1, 15, 16, 17, 0, 100, 333]
    nb, tab = tables_for(lens, bs, gen)
    kp, vp, ks, vs = make_cache(gen, nb, h, bs, d)
    loc = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32) + 2
    n = int(loc[-1])
    ko = torch.full((n + 5, h, d), 7.0, dtype=dtype, device=cuda_device)
    vo = ko.clone()
    flag = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    ops.read_cache_fp8(ko, vo, kp, vp, ks, vs, tab, loc.to(cuda_device), flag)
    assert flag.item() == 0
    for o, pool, sc in ((ko, kp, ks), (vo, vp, vs)):
        assert (o[:2] == 7).all() and (o[n:] == 7).all()  # rows of no sequence
        for i, m in enumerate(lens):
            c, s = rows_of(pool, sc, tab[i], m)
            # code * scale is one fp32 product, then one rounding to the output type.
            want = (c * s[..., None]).transpose(0, 1)
            got = o[int(loc[i]) : int(loc[i]) + m].double()
            lim = want.abs() * 2.0**-24 + rounded(want, dtype) * (1 + 2.0**-10)
            assert ((got - want).abs() <= lim).all()


def test_read_back_of_pages_outside_the_pool(cuda_device) -> None:  # type: ignore[no-untyped-def]
    gen = torch.Generator(device=cuda_device).manual_seed(3)
    kp, vp, ks, vs = make_cache(gen, 4, 2, 16, 128)
    tab = torch.tensor([[1, 4], [2, -1], [3, 0]], dtype=torch.int32, device=cuda_device)
    loc = torch.tensor([0, 20, 40, 80], dtype=torch.int32, device=cuda_device)  # 40 > 2 blocks
    ko = torch.full((80, 2, 128), 7.0, device=cuda_device)
    vo = ko.clone()
    flag = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    ops.read_cache_fp8(ko, vo, kp, vp, ks, vs, tab, loc, flag)
    assert flag.item() == 1
    for o, pool, sc in ((ko, kp, ks), (vo, vp, vs)):
        val = pool.float() * sc[..., None]
        assert torch.equal(o[:16], val[1].transpose(0, 1)) and (o[16:20] == 0).all()
        assert torch.equal(o[20:36], val[2].transpose(0, 1)) and (o[36:40] == 0).all()
        assert torch.equal(o[56:72], val[0].transpose(0, 1)) and (o[72:] == 0).all()


def test_write_then_read_back_is_within_half_a_step(cuda_device) -> None:  # type: ignore[no-untyped-def]
    gen = torch.Generator(device=cuda_device).manual_seed(9)
    t, h, d = 200, 4, 128
    k = torch.randn(t, h, d, generator=gen, device=cuda_device).bfloat16()
    v = torch.randn(t, h, d, generator=gen, device=cuda_device).bfloat16()
    _, tab = tables_for([t], 16, gen)
    kp, vp, ks, vs = empty_cache(int(tab.max()) + 1, h, 16, d, cuda_device)
    p = torch.arange(t, device=cuda_device)
    slots = tab[0, p // 16].long() * 16 + p % 16
    ops.reshape_and_cache_fp8(k, v, kp, vp, ks, vs, slots)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    loc = torch.tensor([0, t], dtype=torch.int32, device=cuda_device)
    ops.read_cache_fp8(ko, vo, kp, vp, ks, vs, tab, loc)
    for x, o in ((k, ko), (v, vo)):
        x, o = x.double(), o.double()
        step = x.abs().amax(-1, keepdim=True) / 448 * 2.0**-10  # among the subnormals
        lim = torch.maximum(x.abs() * 2.0**-4, step) * (1 + 2.0**-18) + o.abs() * HALF_STEP[k.dtype]
        assert ((o - x).abs() <= lim).all()
