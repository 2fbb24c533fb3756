"""64-bit reference of the 8-bit KV cache and of attention over it (TEST INFRASTRUCTURE only)."""

from __future__ import annotations

import math

import torch

E4M3 = torch.float8_e4m3fn
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def rounded(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Most a value near x moves when it is rounded to dtype (half a step, or half the smallest)."""
    tiny = torch.finfo(dtype).smallest_normal
    return x.abs().clamp_min(tiny) * HALF_STEP[dtype]


def make_cache(gen: torch.Generator, num_blocks: int, hkv: int, bs: int, d: int, spread: float = 0.5,
               ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:  # fmt: skip
    """Codes and scales of Gaussian rows whose magnitudes vary by e^spread."""
    got = []
    for _ in range(2):
        x = torch.randn(num_blocks, hkv, bs, d, generator=gen, device=gen.device)
        s = x.abs().amax(-1) / 448
        mag = torch.exp(spread * torch.randn(num_blocks, hkv, bs, generator=gen, device=gen.device))
        got += [(x / s[..., None]).to(E4M3), s * mag]
    return got[0], got[2], got[1], got[3]


def tables_for(ctx: list[int], bs: int, gen: torch.Generator, spare: int = 3,
               width: int = 0) -> tuple[int, torch.Tensor]:  # fmt: skip
    """Blocks in the pool and int32 tables of shuffled distinct blocks, padded with 0."""
    need = [-(-n // bs) for n in ctx]
    total = sum(need) + spare
    perm = torch.randperm(total, generator=gen, device=gen.device).to(torch.int32)
    t = torch.zeros(len(ctx), max(1, width, *need), dtype=torch.int32, device=gen.device)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = perm[at : at + n]
        at += n
    return total, t


def rows_of(pool: torch.Tensor, scales: torch.Tensor, table: torch.Tensor, n: int
            ) -> tuple[torch.Tensor, torch.Tensor]:  # fmt: skip
    """Codes ``[Hkv, n, D]`` and scales ``[Hkv, n]`` of one sequence in 64 bits."""
    blk = table.long()
    c = pool.view(torch.uint8)[blk].view(E4M3).double().transpose(0, 1).flatten(1, 2)[:, :n]
    return c, scales[blk].double().transpose(0, 1).flatten(1, 2)[:, :n]


def attention(q: torch.Tensor, kc: torch.Tensor, ks: torch.Tensor, vc: torch.Tensor,
              vs: torch.Tensor, scale: float, pos0: int | None, k_half: float = 0.0
              ) -> tuple[torch.Tensor, torch.Tensor]:  # fmt: skip
    """Attention of ``q [n, Hq, D]`` over one sequence, and how far a kernel may be off it.

    ``pos0``: position of the first query (causal), None: every query sees everything. The kernel
    rounds each weight w = p * vs / max(p * vs) to fp16: off by 2^-11 of itself, or by 2^-25 below
    fp16's normal range. Scores are fp32 sums: their error is bounded by (D + 2) 2^-23 sum|q k|,
    and by ``k_half`` sum|q k| more where K's values are rounded to a half step of ``k_half``.
    V's values are rounded with it too. A score error e moves a weight by the factor exp(2 e).
    """
    n, hq, d = q.shape
    hkv, ctx, _ = kc.shape
    g = hq // hkv
    qd = q.double().view(n, hkv, g, d)
    k, v = kc * ks[..., None], vc * vs[..., None]
    s = torch.einsum("nhgd,hkd->nhgk", qd, k) * scale
    mass = torch.einsum("nhgd,hkd->nhgk", qd.abs(), k.abs()) * abs(scale)
    if pos0 is not None:
        see = (torch.arange(ctx, device=q.device)[None, :]
               <= pos0 + torch.arange(n, device=q.device)[:, None])  # fmt: skip
        s = s.masked_fill(~see[:, None, None, :], -math.inf)
        mass = mass.masked_fill(~see[:, None, None, :], 0.0)
    m = s.amax(-1, keepdim=True).clamp_min(-1e300)
    p = torch.exp(s - m)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    out = torch.einsum("nhgk,hkd->nhgd", p, v)
    weight = torch.einsum("nhgk,hkd->nhgd", p, v.abs())
    top = (p * vs[None, :, None, :]).amax(-1, keepdim=True)
    tail = 2.0**-25 * top * vc.abs().sum(1)[None, :, None, :] * 2.0
    err = mass.amax(-1, keepdim=True) * ((d + 2) * 2.0**-23 + k_half)
    off = weight * (2.0**-11 + k_half + torch.expm1(2 * err) + 2.0**-19) + tail
    off = off + rounded(out, q.dtype)
    return out.reshape(n, hq, d), off.reshape(n, hq, d)
