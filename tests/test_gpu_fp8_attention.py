"""Decode and chunked-prefill attention over the 8-bit KV cache (GPU).

Compared with 64-bit attention over the very values the cache holds; ``fp8_reference.attention``
derives how far a kernel may be off.
"""

from __future__ import annotations

import pytest
import torch

from tests.fp8_reference import E4M3, HALF_STEP, attention, make_cache, rows_of, tables_for
from tokenserve_b200 import ops

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32


def spoil_unused(cache, tab, ctx, bs):  # type: ignore[no-untyped-def]
    """NaN codes and NaN or huge scales in every slot that holds no token."""
    kp, vp, ks, vs = cache
    used = torch.zeros(kp.shape[0], bs, dtype=torch.bool, device=kp.device)
    for i, n in enumerate(ctx):
        for j in range(-(-n // bs)):
            used[int(tab[i, j]), : min(bs, n - j * bs)] = True
    free = ~used[:, None, :].expand(ks.shape)
    for pool, sc, bad in ((kp, ks, float("nan")), (vp, vs, 3e38)):
        pool.view(torch.uint8)[free] = 0x7F
        sc[free] = bad
        sc[-1][free[-1]] = float("inf")


def decode(q, cache, tab, ctx, scale=None, ws=None, reuse=False, out=None):  # type: ignore[no-untyped-def]
    kp, vp, ks, vs = cache
    b, hq, d = q.shape
    n = ops.decode_workspace_size(b, hq, kp.shape[1], d, tab.shape[1], kp.shape[2], q.dtype)
    ws = torch.empty(max(n, 256), dtype=torch.uint8, device=q.device) if ws is None else ws
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device=q.device) if out is None else out
    ops.paged_decode_fp8(out, q, kp, vp, ks, vs, tab, ctx, scale or d**-0.5, ws, reuse)
    return out


def check_decode(out, q, cache, tab, ctx, scale=None):  # type: ignore[no-untyped-def]
    kp, vp, ks, vs = cache
    for i, n in enumerate(ctx):
        if n == 0:
            assert (out[i] == 0).all()
            continue
        want, off = attention(q[i : i + 1], *rows_of(kp, ks, tab[i], n), *rows_of(vp, vs, tab[i], n),
                              scale or q.shape[-1] ** -0.5, None)  # fmt: skip
        bad = (out[i : i + 1].double() - want).abs() - off
        assert (bad <= 0).all(), (i, n, float(bad.max()))


RAGGED = [1, 0, 15, 16, 17, 31, 33, 255, 256, 700, 1025, 2000]


@pytest.mark.parametrize(
    ("dtype", "hq", "hkv", "d", "bs"),
    [(BF, 32, 8, 128, 16), (FH, 64, 8, 128, 16), (BF, 8, 8, 64, 16), (FH, 28, 4, 64, 16),
     (BF, 16, 1, 128, 16), (BF, 40, 8, 128, 16), (FH, 9, 1, 128, 16),
     (F32, 4, 2, 64, 16), (BF, 34, 2, 128, 16), (FH, 4, 2, 256, 16), (BF, 4, 2, 128, 8),
     (F32, 6, 3, 32, 7)],
)  # fmt: skip
def test_decode_over_ragged_contexts(cuda_device, dtype, hq, hkv, d, bs) -> None:  # type: ignore[no-untyped-def]
    gen = torch.Generator(device=cuda_device).manual_seed(hq * d)
    nb, tab = tables_for(RAGGED, bs, gen, width=140)
    cache = make_cache(gen, nb, hkv, bs, d)
    spoil_unused(cache, tab, RAGGED, bs)
    q = torch.randn(len(RAGGED), hq, d, generator=gen, device=cuda_device).to(dtype)
    ctx = torch.tensor(RAGGED, dtype=torch.int32, device=cuda_device)
    check_decode(decode(q, cache, tab, ctx), q, cache, tab, RAGGED)


@pytest.mark.parametrize("lens", [[1], [5000], [16] * 300, [9000, 3, 0, 4097]])
def test_decode_splits(cuda_device, lens) -> None:  # type: ignore[no-untyped-def]
    """One short and one long sequence, many one-block ones, and a mix: every way work is split."""
    gen = torch.Generator(device=cuda_device).manual_seed(len(lens))
    nb, tab = tables_for(lens, 16, gen)
    cache = make_cache(gen, nb, 2, 16, 128)
    spoil_unused(cache, tab, lens, 16)
    q = torch.randn(len(lens), 8, 128, generator=gen, device=cuda_device).to(BF)
    ctx = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    check_decode(decode(q, cache, tab, ctx), q, cache, tab, lens)


def test_decode_of_a_large_step_claims_work_dynamically(cuda_device) -> None:  # type: ignore[no-untyped-def]
    gen = torch.Generator(device=cuda_device).manual_seed(2)
    lens = [700 + 37 * i for i in range(96)]
    nb, tab = tables_for(lens, 16, gen)
    cache = make_cache(gen, nb, 8, 16, 128)
    spoil_unused(cache, tab, lens, 16)
    q = torch.randn(len(lens), 32, 128, generator=gen, device=cuda_device).to(BF)
    ctx = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    out = decode(q, cache, tab, ctx)
    check_decode(out, q, cache, tab, lens)
    assert torch.equal(out, decode(q, cache, tab, ctx))  # the claim order changes nothing


@pytest.mark.parametrize("kind", ["big-q", "tiny-q", "sink", "wild-v", "zero-v", "peaked"])
def test_decode_of_uneven_magnitudes(cuda_device, kind) -> None:  # type: ignore[no-untyped-def]
    """Queries outside fp16's range, a first token that takes nearly all weight with a value
    thousands of times smaller, value rows over many binades, a zero scale."""
    gen = torch.Generator(device=cuda_device).manual_seed(4)
    lens = [1, 40, 333, 2500]
    nb, tab = tables_for(lens, 16, gen)
    kp, vp, ks, vs = make_cache(gen, nb, 2, 16, 128)
    q = torch.randn(len(lens), 8, 128, generator=gen, device=cuda_device).to(BF)
    scale = 128**-0.5
    if kind == "big-q":
        q, scale = (q * 2.0**60).to(BF), scale * 2.0**-60
    elif kind == "tiny-q":
        q, scale = (q * 2.0**-60).to(BF), scale * 2.0**60
    elif kind == "sink":
        for i in range(len(lens)):
            vs[int(tab[i, 0]), :, 0] *= 2.0**-12
            ks[int(tab[i, 0]), :, 0] *= 4
    elif kind == "wild-v":
        vs *= torch.exp2(torch.randint(-20, 21, vs.shape, generator=gen, device=cuda_device).float())
    elif kind == "zero-v":
        vs[:] = 0
    else:
        ks *= 8
    cache = (kp, vp, ks, vs)
    ctx = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    check_decode(decode(q, cache, tab, ctx, scale), q, cache, tab, lens, scale)


def test_decode_plan_reuse_strided_queries_and_shared_workspace(cuda_device) -> None:  # type: ignore[no-untyped-def]
    gen = torch.Generator(device=cuda_device).manual_seed(5)
    lens = [100, 0, 1700, 16]
    nb, tab = tables_for(lens, 16, gen)
    first, second = make_cache(gen, nb, 8, 16, 128), make_cache(gen, nb, 8, 16, 128)
    wide = torch.randn(len(lens), 48 * 128, generator=gen, device=cuda_device).to(BF)
    q = wide[:, 128 : 33 * 128].unflatten(1, (32, 128))
    ctx = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    n = ops.decode_workspace_size(4, 32, 8, 128, tab.shape[1], 16, BF)
    ws = torch.empty(n, dtype=torch.uint8, device=cuda_device)
    for cache, reuse in ((first, False), (second, True), (first, True)):
        check_decode(decode(q, cache, tab, ctx, ws=ws, reuse=reuse), q, cache, tab, lens)


def test_decode_refuses_a_small_or_misaligned_workspace(cuda_device) -> None:  # type: ignore[no-untyped-def]
    gen = torch.Generator(device=cuda_device).manual_seed(15)
    nb, tab = tables_for([40], 16, gen)
    cache = make_cache(gen, nb, 2, 16, 128)
    q = torch.randn(1, 8, 128, generator=gen, device=cuda_device).to(BF)
    ctx = torch.tensor([40], dtype=torch.int32, device=cuda_device)
    n = ops.decode_workspace_size(1, 8, 2, 128, tab.shape[1], 16, BF)
    ws = torch.empty(n + 512, dtype=torch.uint8, device=cuda_device)
    out = torch.full_like(q, 7.0)
    for bad, text in ((ws[:256], "workspace of 256 bytes"), (ws[1 : n + 1], "256-byte aligned")):
        with pytest.raises(ops.KernelError, match=text):
            decode(q, cache, tab, ctx, ws=bad, out=out)
    with pytest.raises(ops.KernelError, match="workspace"):
        ops.paged_decode_fp8(out, q, *cache, tab, ctx, 0.1, None)
    assert (out == 7).all()


def test_a_plan_for_another_batch_is_refused_on_the_device(cuda_device) -> None:  # type: ignore[no-untyped-def]
    gen = torch.Generator(device=cuda_device).manual_seed(16)
    nb, tab = tables_for([40, 60], 16, gen)
    cache = make_cache(gen, nb, 2, 16, 128)
    q = torch.randn(2, 8, 128, generator=gen, device=cuda_device).to(BF)
    ctx = torch.tensor([40, 60], dtype=torch.int32, device=cuda_device)
    n = ops.decode_workspace_size(2, 8, 2, 128, tab.shape[1], 16, BF)
    ws = torch.zeros(n, dtype=torch.uint8, device=cuda_device)
    check_decode(decode(q, cache, tab, ctx, ws=ws), q, cache, tab, [40, 60])
    out = decode(q[:1], cache, tab[:1], ctx[:1], ws=ws, reuse=True)
    assert (out == 7).all() and int(ws[4:8].view(torch.int32)) == 4


@pytest.mark.parametrize("hq", [4, 16])  # 12 and 8 warps a CTA, the latter as over a 16-bit cache
def test_a_plan_for_a_16_bit_cache_is_refused_on_the_device(cuda_device, hq) -> None:  # type: ignore[no-untyped-def]
    gen = torch.Generator(device=cuda_device).manual_seed(17)
    lens = [400, 60]
    nb, tab = tables_for(lens, 16, gen)
    cache = make_cache(gen, nb, 1, 16, 128)
    plain = torch.zeros(2, nb, 1, 16, 128, dtype=BF, device=cuda_device)
    q = torch.randn(2, hq, 128, generator=gen, device=cuda_device).to(BF)
    ctx = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    n = ops.decode_workspace_size(2, hq, 1, 128, tab.shape[1], 16, BF)
    ws = torch.zeros(n, dtype=torch.uint8, device=cuda_device)
    out = torch.full_like(q, 7)
    ops.paged_decode(out, q, plain[0], plain[1], tab, ctx, 0.1, ws)
    assert (out == 0).all()
    out = decode(q, cache, tab, ctx, ws=ws, reuse=True)
    assert (out == 7).all() and int(ws[4:8].view(torch.int32)) == 4
    check_decode(decode(q, cache, tab, ctx, ws=ws), q, cache, tab, lens)
    out = torch.full_like(q, 7)
    ops.paged_decode(out, q, plain[0], plain[1], tab, ctx, 0.1, ws, reuse_plan=True)
    assert (out == 7).all() and int(ws[4:8].view(torch.int32)) == 4


def test_a_nan_row_spoils_its_own_sequence_alone(cuda_device) -> None:  # type: ignore[no-untyped-def]
    gen = torch.Generator(device=cuda_device).manual_seed(6)
    lens = [50, 60, 70, 80]
    nb, tab = tables_for(lens, 16, gen)
    kp, vp, ks, vs = make_cache(gen, nb, 2, 16, 128)
    row = torch.randn(1, 2, 128, generator=gen, device=cuda_device).to(BF)
    bad = row.clone()
    bad[0, :, 5] = float("nan")
    for i, (k, v) in {1: (bad, row), 2: (row, bad)}.items():
        slot = tab[i, 1].long()[None] * 16 + 3
        ops.reshape_and_cache_fp8(k, v, kp, vp, ks, vs, slot)
    q = torch.randn(4, 8, 128, generator=gen, device=cuda_device).to(BF)
    ctx = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    out = decode(q, (kp, vp, ks, vs), tab, ctx)
    assert torch.isnan(out[1]).all() and torch.isnan(out[2]).all()
    check_decode(out[::3], q[::3], (kp, vp, ks, vs), tab[::3], lens[::3])
    qsl = torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32, device=cuda_device)
    pre = torch.zeros_like(q)
    ops.paged_prefill_fp8(pre, q, kp, vp, ks, vs, tab, qsl, ctx, 1, 128**-0.5)
    assert torch.isnan(pre[1]).all() and torch.isnan(pre[2]).all()
    assert torch.isfinite(pre[::3]).all()


# ------------------------------------------------------------------------------ prefill


def prefill(q, cache, tab, qsl, ctx, qmax, scale=None):  # type: ignore[no-untyped-def]
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device=q.device)
    ops.paged_prefill_fp8(out, q, *cache, tab, qsl, ctx, qmax, scale or q.shape[-1] ** -0.5)
    return out


def check_prefill(out, q, cache, tab, chunks, ctx, scale=None, start=0, k_half=2.0**-11):  # type: ignore[no-untyped-def]
    """``k_half``: the tensor-core kernel rounds K's and V's values to fp16 once."""
    kp, vp, ks, vs = cache
    at = start
    for i, (n, c) in enumerate(zip(chunks, ctx, strict=True)):
        rows = slice(at, at + n)
        at += n
        skip = max(0, n - c)  # rows before position 0 see nothing
        assert (out[rows][:skip] == 0).all()
        if n - skip == 0:
            continue
        want, off = attention(q[rows][skip:], *rows_of(kp, ks, tab[i], c),
                              *rows_of(vp, vs, tab[i], c), scale or q.shape[-1] ** -0.5,
                              c - (n - skip), k_half=k_half)  # fmt: skip
        bad = (out[rows][skip:].double() - want).abs() - off
        assert (bad <= 0).all(), (i, n, c, float(bad.max()))


CHUNKS = [1, 17, 0, 128, 33, 200, 64, 5, 300]
CTX = [1, 17, 40, 128, 500, 1111, 64, 2, 300]  # the 8th: a chunk longer than its context


@pytest.mark.parametrize(
    ("dtype", "hq", "hkv", "d", "bs"),
    [(BF, 32, 8, 128, 16), (FH, 16, 2, 128, 16), (BF, 4, 4, 128, 16), (BF, 14, 2, 64, 16),
     (FH, 5, 1, 128, 16), (FH, 16, 1, 64, 16), (BF, 6, 2, 64, 16), (BF, 34, 2, 128, 16),
     (F32, 4, 2, 64, 16), (FH, 4, 2, 256, 16), (BF, 4, 2, 128, 8), (F32, 6, 3, 32, 7)],
)  # fmt: skip
def test_prefill_over_ragged_chunks(cuda_device, dtype, hq, hkv, d, bs) -> None:  # type: ignore[no-untyped-def]
    gen = torch.Generator(device=cuda_device).manual_seed(hq + d)
    nb, tab = tables_for(CTX, bs, gen, width=200)
    cache = make_cache(gen, nb, hkv, bs, d)
    spoil_unused(cache, tab, CTX, bs)
    total = sum(CHUNKS)
    q = torch.randn(total + 9, hq, d, generator=gen, device=cuda_device).to(dtype)
    qsl = torch.tensor([0, *CHUNKS], device=cuda_device).cumsum(0).to(torch.int32) + 4
    ctx = torch.tensor(CTX, dtype=torch.int32, device=cuda_device)
    out = prefill(q, cache, tab, qsl, ctx, max(CHUNKS))
    assert (out[:4] == 7).all() and (out[4 + total :] == 7).all()  # rows of no sequence
    check_prefill(out, q, cache, tab, CHUNKS, CTX, start=4)


def test_prefill_takes_strided_queries_and_a_loose_length_bound(cuda_device) -> None:  # type: ignore[no-untyped-def]
    gen = torch.Generator(device=cuda_device).manual_seed(8)
    chunks, ctxs = [70, 130], [300, 130]
    nb, tab = tables_for(ctxs, 16, gen)
    cache = make_cache(gen, nb, 8, 16, 128)
    wide = torch.randn(200, 48 * 128, generator=gen, device=cuda_device).to(BF)
    q = wide[:, 128 : 33 * 128].unflatten(1, (32, 128))
    qsl = torch.tensor([0, 70, 200], dtype=torch.int32, device=cuda_device)
    ctx = torch.tensor(ctxs, dtype=torch.int32, device=cuda_device)
    out = prefill(q, cache, tab, qsl, ctx, 1000)
    check_prefill(out, q, cache, tab, chunks, ctxs)


@pytest.mark.parametrize("kind", ["big-q", "tiny-q", "sink", "wild-v", "wild-k", "zero-v", "peaked"])
def test_prefill_of_uneven_magnitudes(cuda_device, kind) -> None:  # type: ignore[no-untyped-def]
    gen = torch.Generator(device=cuda_device).manual_seed(10)
    chunks, ctxs = [40, 150], [900, 150]
    nb, tab = tables_for(ctxs, 16, gen)
    kp, vp, ks, vs = make_cache(gen, nb, 2, 16, 128)
    q = torch.randn(190, 8, 128, generator=gen, device=cuda_device).to(BF)
    scale = 128**-0.5
    if kind == "big-q":
        q, scale = (q * 2.0**60).to(BF), scale * 2.0**-60
    elif kind == "tiny-q":
        q, scale = (q * 2.0**-60).to(BF), scale * 2.0**60
    elif kind == "sink":
        for i in range(2):
            vs[int(tab[i, 0]), :, 0] *= 2.0**-12
            ks[int(tab[i, 0]), :, 0] *= 4
    elif kind == "wild-v":
        vs *= 2.0 ** torch.randint(-3, 4, vs.shape, generator=gen, device=cuda_device).float()
    elif kind == "wild-k":  # whole tiles of other magnitudes
        ks *= 2.0 ** torch.randint(-40, 1, (ks.shape[0], 1, 1), generator=gen,
                                   device=cuda_device).float()  # fmt: skip
    elif kind == "zero-v":
        vs[:] = 0
    else:
        ks *= 8
    cache = (kp, vp, ks, vs)
    qsl = torch.tensor([0, 40, 190], dtype=torch.int32, device=cuda_device)
    ctx = torch.tensor(ctxs, dtype=torch.int32, device=cuda_device)
    out = prefill(q, cache, tab, qsl, ctx, 150, scale)
    check_prefill(out, q, cache, tab, chunks, ctxs, scale)


@pytest.mark.parametrize(("dtype", "hq", "d"), [(BF, 8, 128), (FH, 8, 64), (F32, 4, 64)])
@pytest.mark.parametrize("which", ["key", "value"])
def test_a_nan_row_reaches_only_the_queries_that_see_it(cuda_device, dtype, hq, d, which) -> None:  # type: ignore[no-untyped-def]
    """One position of a chunk holds a NaN, for each place of it in the column groups."""
    gen = torch.Generator(device=cuda_device).manual_seed(13)
    chunk, ctx = 100, 230
    qsl = torch.tensor([0, chunk], dtype=torch.int32, device=cuda_device)
    cl = torch.tensor([ctx], dtype=torch.int32, device=cuda_device)
    nb, tab = tables_for([ctx], 16, gen)
    q = torch.randn(chunk, hq, d, generator=gen, device=cuda_device).to(dtype)
    for at in (130, 131, 134, 159, 160, 191, 192, 200, 229):
        kp, vp, ks, vs = make_cache(gen, nb, 2, 16, d)
        row = torch.randn(1, 2, d, generator=gen, device=cuda_device).to(dtype)
        bad = row.clone()
        bad[0, :, 5] = float("nan")
        slot = tab[0, at // 16].long()[None] * 16 + at % 16
        ops.reshape_and_cache_fp8(*((bad, row) if which == "key" else (row, bad)), kp, vp, ks, vs,
                                  slot)  # fmt: skip
        out = prefill(q, (kp, vp, ks, vs), tab, qsl, cl, chunk)
        first = at - (ctx - chunk)  # the first query that sees it
        assert torch.isnan(out[first:]).all()
        if first:
            check_prefill(out[:first], q[:first], (kp, vp, ks, vs), tab, [first], [at])


@pytest.mark.parametrize(("dtype", "hq", "d"), [(BF, 8, 128), (FH, 4, 64), (F32, 4, 64)])
@pytest.mark.parametrize("bad", [-1, -(2**31), 2**31 - 1, 40])
def test_pages_outside_the_pool_are_skipped(cuda_device, dtype, hq, d, bad) -> None:  # type: ignore[no-untyped-def]
    """Attention over the other blocks alone: their tokens' positions stay where they were, which only
    the causal mask uses (the chunk lies in a block after the skipped ones)."""
    gen = torch.Generator(device=cuda_device).manual_seed(14)
    ctx = 150
    nb, tab = tables_for([ctx, ctx], 16, gen, spare=40 - 20)
    kp, vp, ks, vs = make_cache(gen, nb, 2, 16, d)
    cache = (kp, vp, ks, vs)
    assert nb == 40
    broken, kept = tab.clone(), {0: [0, 1, 2, 4, 5, 7, 8, 9], 1: [5, 6, 8, 9]}
    for i, blocks in kept.items():
        for j in range(10):
            if j not in blocks:
                broken[i, j] = bad
    lens = [len(b) * 16 - 10 for b in kept.values()]  # the last block holds 6 tokens
    whole = torch.zeros_like(tab)
    for i, blocks in kept.items():
        whole[i, : len(blocks)] = tab[i, blocks]
    cl = torch.tensor([ctx, ctx], dtype=torch.int32, device=cuda_device)
    q = torch.randn(2, hq, d, generator=gen, device=cuda_device).to(dtype)
    check_decode(decode(q, cache, broken, cl), q, cache, whole, lens)
    chunks = [4, 6]
    qsl = torch.tensor([0, 4, 10], dtype=torch.int32, device=cuda_device)
    q = torch.randn(10, hq, d, generator=gen, device=cuda_device).to(dtype)
    out = prefill(q, cache, broken, qsl, cl, 6)
    check_prefill(out, q, cache, whole, chunks, lens)


# ------------------------------------------------------------------------------ together


def test_a_model_step_over_the_cache(cuda_device) -> None:  # type: ignore[no-untyped-def]
    """Prompt chunks written and attended, then decode steps, as a model's layer runs them; the
    attention agrees with 64-bit attention over what read_cache_fp8 returns."""
    gen = torch.Generator(device=cuda_device).manual_seed(11)
    hq, hkv, d, bs = 8, 2, 128, 16
    prompts, steps = [33, 7, 100], 3
    final = [p + steps for p in prompts]
    nb, tab = tables_for(final, bs, gen)
    kp = torch.zeros(nb, hkv, bs, d, dtype=torch.uint8, device=cuda_device).view(E4M3)
    vp, ks = kp.clone(), torch.zeros(nb, hkv, bs, device=cuda_device)
    vs = ks.clone()
    cache = (kp, vp, ks, vs)
    inv = (500000.0 ** (-torch.arange(d // 2, device=cuda_device) / (d // 2))).float()

    def write(positions):  # type: ignore[no-untyped-def]
        seq = torch.cat([torch.full((len(p),), i) for i, p in enumerate(positions)]).to(cuda_device)
        pos = torch.cat(positions).to(cuda_device)
        slots = tab[seq, pos // bs].long() * bs + pos % bs
        qkv = torch.randn(len(pos), (hq + 2 * hkv) * d, generator=gen, device=cuda_device).to(BF)
        q = torch.empty(len(pos), hq, d, dtype=BF, device=cuda_device)
        ops.rotary_and_cache(qkv, q, kp, vp, slots, pos, inv, hq, hkv, key_scales=ks,
                             value_scales=vs)  # fmt: skip
        return q

    q = write([torch.arange(p) for p in prompts])
    qsl = torch.tensor([0, *prompts], device=cuda_device).cumsum(0).to(torch.int32)
    ctx = torch.tensor(prompts, dtype=torch.int32, device=cuda_device)
    out = prefill(q, cache, tab, qsl, ctx, max(prompts))
    check_prefill(out, q, cache, tab, prompts, prompts)
    for s in range(steps):
        lens = [p + s + 1 for p in prompts]
        q = write([torch.tensor([n - 1]) for n in lens])
        out = decode(q, cache, tab, torch.tensor(lens, dtype=torch.int32, device=cuda_device))
        check_decode(out, q, cache, tab, lens)
    loc = torch.tensor([0, *final], device=cuda_device).cumsum(0).to(torch.int32)
    ko = torch.empty(int(loc[-1]), hkv, d, device=cuda_device)
    vo = torch.empty_like(ko)
    ops.read_cache_fp8(ko, vo, *cache, tab, loc)
    for i, n in enumerate(final):
        k, v = ko[loc[i] : loc[i + 1]].double(), vo[loc[i] : loc[i + 1]].double()
        p = torch.softmax(torch.einsum("hd,khd->hk", q[i].double(),
                                       k.repeat_interleave(hq // hkv, 1)) * d**-0.5, -1)  # fmt: skip
        want = torch.einsum("hk,khd->hd", p, v.repeat_interleave(hq // hkv, 1))
        _, off = attention(q[i : i + 1], *rows_of(kp, ks, tab[i], n), *rows_of(vp, vs, tab[i], n),
                           d**-0.5, None)  # fmt: skip
        assert ((out[i].double() - want).abs() <= off[0] + 2.0**-23 * want.abs()).all()


@pytest.mark.parametrize("dtype", [BF, F32])  # tensor cores, CUDA cores
def test_blocks_whose_offsets_pass_32_bits(cuda_device, dtype) -> None:  # type: ignore[no-untyped-def]
    """Every operator on the last blocks of pools of 4.6 GB each, and on block 0."""
    gen = torch.Generator(device=cuda_device).manual_seed(13)
    nb, hq, hkv, bs, d, n = 140_000, 32, 16, 16, 128, 150
    assert (nb - 20) * hkv * bs * d > 2**32
    kp = torch.empty(nb, hkv, bs, d, dtype=torch.uint8, device=cuda_device).view(E4M3)
    vp = torch.empty_like(kp)
    ks = torch.empty(nb, hkv, bs, device=cuda_device)
    vs = torch.empty_like(ks)
    cache = (kp, vp, ks, vs)
    last = nb - 1 - torch.arange(9, device=cuda_device)
    tab = torch.cat([last, torch.zeros(1, device=cuda_device)]).to(torch.int32)[None]
    pos = torch.arange(n, device=cuda_device)
    slots = tab[0, pos // bs].long() * bs + pos % bs
    k = torch.randn(n, hkv, d, generator=gen, device=cuda_device).to(dtype)
    v = torch.randn(n, hkv, d, generator=gen, device=cuda_device).to(dtype)
    half = n // 2
    ops.reshape_and_cache_fp8(k[:half], v[:half], kp, vp, ks, vs, slots[:half])
    q = torch.randn(n, hq, d, generator=gen, device=cuda_device).to(dtype)
    qkv = torch.cat([q[half:].flatten(1), k[half:].flatten(1), v[half:].flatten(1)], 1)
    still = torch.zeros(d // 2, device=cuda_device)  # nothing turns
    ops.rotary_and_cache(qkv, torch.empty_like(q[half:]), kp, vp, slots[half:], pos[half:], still, hq,
                         hkv, key_scales=ks, value_scales=vs)  # fmt: skip
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    loc = torch.tensor([0, n], dtype=torch.int32, device=cuda_device)
    ops.read_cache_fp8(ko, vo, *cache, tab, loc)
    for x, o in ((k, ko), (v, vo)):
        # Half a step: 2^-4 of the value, or of the smallest normal (2^-6 of a code, 448 the row's
        # largest); fp32 steps of the scale and the quotient; the output's own rounding.
        x, o = x.double(), o.double()
        least = x.abs().amax(-1, keepdim=True) / 448 * 2.0**-6
        lim = torch.maximum(x.abs(), least) * 2.0**-4 * (1 + 2.0**-18) + o.abs() * HALF_STEP[dtype]
        assert ((o - x).abs() <= lim).all()
    ctx = torch.tensor([n], dtype=torch.int32, device=cuda_device)
    check_decode(decode(q[-1:], cache, tab, ctx), q[-1:], cache, tab, [n])
    check_prefill(prefill(q, cache, tab, loc, ctx, n), q, cache, tab, [n], [n])


def test_captured_step_replays_on_new_inputs_on_another_stream(cuda_device) -> None:  # type: ignore[no-untyped-def]
    gen = torch.Generator(device=cuda_device).manual_seed(12)
    lens = [17, 300, 64]
    nb, tab = tables_for(lens, 16, gen)
    cache = make_cache(gen, nb, 2, 16, 128)
    ctx = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    qkv = torch.zeros(3, 12 * 128, dtype=BF, device=cuda_device)
    pos = torch.tensor([n - 1 for n in lens], device=cuda_device)
    slots = tab[torch.arange(3, device=cuda_device), pos // 16].long() * 16 + pos % 16
    inv = torch.rand(64, device=cuda_device)
    q = torch.zeros(3, 8, 128, dtype=BF, device=cuda_device)
    out, pre = torch.zeros_like(q), torch.zeros_like(q)
    qsl = torch.arange(4, dtype=torch.int32, device=cuda_device)
    n = ops.decode_workspace_size(3, 8, 2, 128, tab.shape[1], 16, BF)
    ws = torch.empty(n, dtype=torch.uint8, device=cuda_device)

    def step():  # type: ignore[no-untyped-def]
        ops.rotary_and_cache(qkv, q, cache[0], cache[1], slots, pos, inv, 8, 2,
                             key_scales=cache[2], value_scales=cache[3])  # fmt: skip
        ops.paged_decode_fp8(out, q, *cache, tab, ctx, 128**-0.5, ws)
        ops.paged_prefill_fp8(pre, q, *cache, tab, qsl, ctx, 1, 128**-0.5)

    side = torch.cuda.Stream(device=cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(2):
        qkv.copy_(torch.randn(qkv.shape, generator=gen, device=cuda_device))
        graph.replay()
        torch.cuda.synchronize()
        check_decode(out, q, cache, tab, lens)
        check_prefill(pre, q, cache, tab, [1, 1, 1], lens)
