"""The operators of the 8-bit paged KV cache, as cases to measure.

Five operators that work on one cache: writing new K/V rows into it (``append``), rotary
positions fused with that write (``rotary``), reading rows back (``read``), and the decode and
chunked-prefill attention over it (``decode``, ``prefill``). With ``own`` false, :func:`run`
computes them with elementary torch operations in 32 bits; with ``own`` true it calls
``tokenserve_b200.ops``.

The cache holds, per layer and for K and V each, e4m3 codes ``[blocks, kv_heads, block, dim]`` and
one float32 scale per (token, KV head) ``[blocks, kv_heads, block]``. A row ``x`` is stored as
``scale = max(amax|x| / 448, 2^-126)`` and ``code = e4m3(x / scale)``; it stands for
``code * scale``.
"""

import math

import numpy as np
import torch

own = False

BLOCK = 16
E4M3_MAX = 448.0
MIN_SCALE = 2.0**-126
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ESIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------------------ cases


def listed():
    return [
        # One decode step's new tokens of 256 sequences (Llama-3-8B heads): latency counts.
        {"name": "append-decode", "op": "append", "dtype": "bf16", "tokens": 256, "run": 1,
         "hkv": 8, "d": 128, "strided": True, "pad": 7},
        # A prefill round of 64 sequences x 512 tokens: HBM-bound.
        {"name": "append-prefill", "op": "append", "dtype": "bf16", "tokens": 32768, "run": 512,
         "hkv": 8, "d": 128, "strided": True, "pad": 0},
        # Decode step of 256 sequences: rotary positions scaled for long contexts, then the write.
        {"name": "rotary-decode", "op": "rotary", "dtype": "bf16", "tokens": 256, "run": 1,
         "hq": 32, "hkv": 8, "d": 128, "rd": 128, "interleaved": False, "scaling": "wavelength",
         "quant": True, "maxpos": 131072},
        # A long prompt's chunk round into the 8-bit cache, odd token count.
        {"name": "rotary-prefill", "op": "rotary", "dtype": "bf16", "tokens": 16381, "run": 512,
         "hq": 32, "hkv": 8, "d": 128, "rd": 128, "interleaved": False, "scaling": "wavelength",
         "quant": True, "maxpos": 131072},
        # Interleaved pairs on half of each head, stretched positions, cache in the model's type.
        {"name": "rotary-partial", "op": "rotary", "dtype": "f16", "tokens": 4099, "run": 100,
         "hq": 64, "hkv": 8, "d": 128, "rd": 64, "interleaved": True, "scaling": "factor",
         "quant": False, "maxpos": 32768},
        # One sequence's context read back (handing a cached prefix to another process).
        {"name": "read-one", "op": "read", "dtype": "bf16", "seqs": 1, "median": 1500,
         "sigma": 0.0, "lo": 1, "hi": 8192, "hkv": 8, "d": 128},
        # 64 sequences' contexts of ragged lengths.
        {"name": "read-many", "op": "read", "dtype": "f16", "seqs": 64, "median": 1024,
         "sigma": 0.7, "lo": 1, "hi": 8192, "hkv": 8, "d": 128},
        # One sequence decoding: the latency of a single user.
        {"name": "decode-one", "op": "decode", "dtype": "bf16", "batch": 1, "median": 1000,
         "sigma": 0.0, "lo": 1, "hi": 8192, "hq": 32, "hkv": 8, "d": 128},
        # The decode benchmark's batch: 256 sequences, log-normal contexts (Llama-3-8B heads).
        {"name": "decode-256", "op": "decode", "dtype": "bf16", "batch": 256, "median": 1024,
         "sigma": 1.0, "lo": 16, "hi": 8192, "hq": 32, "hkv": 8, "d": 128},
        # Long contexts at Llama-3-70B heads, fp16.
        {"name": "decode-long", "op": "decode", "dtype": "f16", "batch": 64, "median": 4096,
         "sigma": 1.0, "lo": 16, "hi": 32768, "hq": 64, "hkv": 8, "d": 128},
        # One sequence's 512-token chunk over a 1024-token cached prefix.
        {"name": "prefill-one", "op": "prefill", "dtype": "bf16", "seqs": 1, "qlo": 512,
         "qhi": 512, "plo": 1024, "phi": 1024, "hq": 32, "hkv": 8, "d": 128},
        # The prefill benchmark's round: 64 sequences, ragged chunks over ragged cached prefixes.
        {"name": "prefill-64", "op": "prefill", "dtype": "bf16", "seqs": 64, "qlo": 257,
         "qhi": 512, "plo": 900, "phi": 1600, "hq": 32, "hkv": 8, "d": 128},
    ]  # fmt: skip


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "rotary", "read", "decode", "prefill"])
    dtype = rng.choice(["bf16", "f16"])
    d = rng.choice([64, 128])
    hkv = rng.choice([1, 2, 4, 8])
    if op == "append":
        return {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"]),
                "tokens": _log_int(rng, 1, 16384), "run": rng.choice([1, 100, 512]),
                "hkv": hkv, "d": d,
                "strided": rng.random() < 0.5, "pad": rng.choice([0, 3, 7])}  # fmt: skip
    g = rng.choice([1, 2, 4, 5, 7, 8, 16])
    if op == "rotary":
        return {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"]),
                "tokens": _log_int(rng, 1, 8192), "run": rng.choice([1, 100, 512]),
                "hq": hkv * min(g, 8), "hkv": hkv, "d": d,
                "rd": rng.choice([d, d // 2]), "interleaved": rng.random() < 0.5,
                "scaling": rng.choice(["none", "wavelength", "factor"]),
                "quant": rng.random() < 0.7, "maxpos": _log_int(rng, 64, 131072)}  # fmt: skip
    if op == "read":
        return {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"]),
                "seqs": _log_int(rng, 1, 64), "median": _log_int(rng, 8, 1024),
                "sigma": rng.choice([0.0, 0.5, 1.0]), "lo": 1, "hi": 4096, "hkv": hkv,
                "d": d}  # fmt: skip
    if op == "decode":
        batch = _log_int(rng, 1, 256)
        return {"op": op, "dtype": dtype, "batch": batch,
                "median": _log_int(rng, 8, min(8192, 262144 // batch)),
                "sigma": rng.choice([0.0, 0.5, 1.0]), "lo": rng.choice([0, 1, 16]),
                "hi": min(16384, 2097152 // batch), "hq": hkv * g, "hkv": hkv, "d": d}  # fmt: skip
    seqs = _log_int(rng, 1, 32)
    qhi = _log_int(rng, 1, 1024)
    phi = _log_int(rng, 1, 2048)
    return {"op": op, "dtype": dtype, "seqs": seqs, "qlo": max(1, qhi // 3), "qhi": qhi,
            "plo": phi // 3, "phi": phi, "hq": min(32, hkv * g) // hkv * hkv, "hkv": hkv,
            "d": d}  # fmt: skip


def _lens(case):
    """Sequence lengths: fixed by the case alone, so every seed has the same work."""
    r = np.random.default_rng(case.get("batch", case.get("seqs", 1)) * 31 + 5)
    if case["op"] == "prefill":
        q = r.integers(case["qlo"], case["qhi"], case["seqs"], endpoint=True)
        p = r.integers(case["plo"], case["phi"], case["seqs"], endpoint=True)
        return q.astype(np.int64), p.astype(np.int64)
    n = case["batch"] if case["op"] == "decode" else case["seqs"]
    z = np.exp(math.log(case["median"]) + case["sigma"] * r.standard_normal(n))
    return np.clip(np.round(z), case["lo"], case["hi"]).astype(np.int64)


def work(case):
    op, d, hkv, es = case["op"], case["d"], case["hkv"], ESIZE[case["dtype"]]
    row = hkv * (d + 4) * 2  # one token's K and V in the cache: codes and scales
    if op == "append":
        t = case["tokens"] - (-(-case["tokens"] // case["pad"]) if case["pad"] else 0)
        return {"bytes": t * (hkv * d * es * 2 + row) + case["tokens"] * 8,
                "flops": t * hkv * d * 6}  # fmt: skip
    if op == "rotary":
        t, hq = case["tokens"], case["hq"]
        kv = row if case["quant"] else 2 * hkv * d * es
        return {"bytes": t * ((hq + 2 * hkv) * d * es + hq * d * es + kv + 16),
                "flops": t * (hq + hkv) * case["rd"] * 3}  # fmt: skip
    if op == "read":
        t = int(_lens(case).sum())
        return {"bytes": t * (row + hkv * d * es * 2), "flops": t * hkv * d * 2}
    hq = case["hq"]
    if op == "decode":
        n = _lens(case)
        t = int(n.sum())
        return {"bytes": t * row + len(n) * hq * d * es * 2 + int(((n + 15) // 16).sum()) * 4,
                "flops": 4 * hq * d * t}  # fmt: skip
    q, p = _lens(case)
    seen = int((q * p + q * (q + 1) // 2).sum())
    return {"bytes": int((q + p).sum()) * row + int(q.sum()) * hq * d * es * 2,
            "flops": 4 * hq * d * seen}  # fmt: skip


# ------------------------------------------------------------------------------ inputs


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _inv_freq(case):
    """Rotary frequencies and the factor on cos and sin. "wavelength": long wavelengths are
    stretched 8 times, short ones kept, a ramp between (contexts beyond 8192); "factor": every
    frequency a quarter, cos and sin scaled up by a mild factor."""
    half = case["rd"] // 2
    base = 500000.0 if case["scaling"] == "wavelength" else 10000.0
    f = base ** (-np.arange(half, dtype=np.float64) / half)
    if case["scaling"] == "wavelength":
        turns = 8192.0 * f / (2 * math.pi)
        keep = np.clip((turns - 1.0) / 3.0, 0.0, 1.0)
        f = f * (keep + (1.0 - keep) / 8.0)
    if case["scaling"] == "factor":
        f = f / 4.0
    mscale = 0.1 * math.log(4.0) + 1.0 if case["scaling"] == "factor" else 1.0
    return torch.from_numpy(f.astype(np.float32)).cuda(), mscale


def _rows(g, n, h, d, dtype):
    """Rows as a projection leaves them: per-head magnitudes apart, a few large channels."""
    x = torch.randn(n, h, d, generator=g, device="cuda")
    mag = torch.exp(0.5 * torch.randn(n, h, 1, generator=g, device="cuda"))
    big = 1.0 + 3.0 * (torch.rand(1, h, d, generator=g, device="cuda") < 0.03)
    return (x * mag * big * 0.7).to(dtype)


def _cache(g, blocks, hkv, d):
    """A filled cache: codes of rows of varying magnitude, and their scales."""
    pools = []
    for _ in range(2):
        x = torch.randn(blocks, hkv, BLOCK, d, generator=g, device="cuda")
        s = x.abs().amax(-1) / E4M3_MAX
        codes = (x / s[..., None]).to(torch.float8_e4m3fn)
        mag = torch.exp(0.4 * torch.randn(blocks, hkv, BLOCK, generator=g, device="cuda"))
        pools += [codes, s * mag]
        del x
    return {"kp": pools[0], "ks": pools[1], "vp": pools[2], "vs": pools[3]}


def _tables(r, ctx, spare=8):
    need = -(-ctx // BLOCK)
    blocks = int(need.sum()) + spare
    perm = r.permutation(blocks).astype(np.int32)
    t = np.zeros((len(ctx), max(1, int(need.max()))), np.int32)
    off = 0
    for i, n in enumerate(need.tolist()):
        t[i, :n] = perm[off : off + n]
        off += n
    return blocks, torch.from_numpy(t).cuda()


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()


def prepare(case, seed):
    g, r = _gen(seed), np.random.default_rng(int(seed))
    dt, d, hkv = DTYPES[case["dtype"]], case["d"], case["hkv"]
    s = {"case": case}
    if case["op"] in ("append", "rotary"):
        # Sequences of `run` new tokens each, every sequence in blocks of its own anywhere in
        # the pool: run 1 is a decode step (any place in its last block), more a prefill chunk.
        t, run = case["tokens"], case["run"]
        seqs, width = -(-t // run), -(-run // BLOCK)
        blocks = seqs * width + 4
        home = r.permutation(blocks)[: seqs * width].reshape(seqs, width)
        seq, at = np.divmod(np.arange(t), run)
        off = r.integers(0, BLOCK, t) if run == 1 else at % BLOCK
        slots = (home[seq, at // BLOCK] * BLOCK + off).astype(np.int64)
        if case.get("pad"):
            slots[:: case["pad"]] = -1
        s["slots"] = torch.from_numpy(slots).cuda()
        quant = case.get("quant", True)
        shape = (blocks, hkv, BLOCK, d)
        for p in ("kp", "vp"):
            pool = torch.zeros(shape, dtype=torch.uint8 if quant else dt, device="cuda")
            s[p] = pool.view(torch.float8_e4m3fn) if quant else pool
        for p in ("ks", "vs"):
            s[p] = torch.full(shape[:3], MIN_SCALE, device="cuda") if quant else None
    if case["op"] == "append":
        if case["strided"]:  # K and V inside one fused projection
            kv = _rows(g, t, 2 * hkv, d, dt)
            s["k"], s["v"] = kv[:, :hkv], kv[:, hkv:]
        else:
            s["k"], s["v"] = _rows(g, t, hkv, d, dt), _rows(g, t, hkv, d, dt)
    elif case["op"] == "rotary":
        hq = case["hq"]
        s["qkv"] = _rows(g, t, hq + 2 * hkv, d, dt).view(t, -1)
        first = r.integers(0, max(1, case["maxpos"] - run + 1), seqs)
        s["pos"] = torch.from_numpy((first[seq] + at).astype(np.int64)).cuda()
        s["inv_freq"], s["mscale"] = _inv_freq(case)
        s["q_out"] = torch.zeros(t, hq, d, dtype=dt, device="cuda")
    elif case["op"] == "read":
        n = _lens(case)
        blocks, s["tables"] = _tables(r, n)
        s.update(_cache(g, blocks, hkv, d))
        loc = np.concatenate([[0], np.cumsum(n)])
        s["loc"] = _i32(loc)
        s["k_out"] = torch.zeros(int(loc[-1]), hkv, d, dtype=dt, device="cuda")
        s["v_out"] = torch.zeros_like(s["k_out"])
    elif case["op"] == "decode":
        n = _lens(case)
        blocks, s["tables"] = _tables(r, n)
        s.update(_cache(g, blocks, hkv, d))
        s["ctx"] = _i32(n)
        s["q"] = torch.randn(len(n), case["hq"], d, generator=g, device="cuda").to(dt)
        s["out"] = torch.zeros_like(s["q"])
    else:
        q, p = _lens(case)
        blocks, s["tables"] = _tables(r, q + p)
        s.update(_cache(g, blocks, hkv, d))
        s["ctx"], s["qmax"] = _i32(q + p), int(q.max())
        loc = np.concatenate([[0], np.cumsum(q)])
        s["qsl"] = _i32(loc)
        s["q"] = torch.randn(int(loc[-1]), case["hq"], d, generator=g, device="cuda").to(dt)
        s["out"] = torch.zeros_like(s["q"])
    return s


# ------------------------------------------------------------------------------ one pass


def run(state):
    if own:
        return _run_own(state)
    return {"append": _append, "rotary": _rotary, "read": _read, "decode": _decode,
            "prefill": _prefill}[state["case"]["op"]](state)  # fmt: skip


def _written(s):
    """What a write leaves: both pools, with their scales where the cache is 8-bit."""
    return {k: s[k] for k in ("kp", "vp", "ks", "vs", "q_out") if s.get(k) is not None}


def _run_own(s):
    from tokenserve_b200 import ops

    case = s["case"]
    op, d = case["op"], case["d"]
    cache = (s["kp"], s["vp"], s["ks"], s["vs"])
    if op == "append":
        ops.reshape_and_cache_fp8(s["k"], s["v"], *cache, s["slots"])
        return _written(s)
    if op == "rotary":
        ops.rotary_and_cache(s["qkv"], s["q_out"], s["kp"], s["vp"], s["slots"], s["pos"],
                             s["inv_freq"], case["hq"], case["hkv"], key_scales=s["ks"],
                             value_scales=s["vs"], interleaved=case["interleaved"],
                             attention_scaling=s["mscale"])  # fmt: skip
        return _written(s)
    if op == "read":
        ops.read_cache_fp8(s["k_out"], s["v_out"], *cache, s["tables"], s["loc"])
        return s["k_out"], s["v_out"]
    if op == "decode":
        if "ws" not in s:  # kept by the program that owns the cache, as its model runner does
            n = ops.decode_workspace_size(s["q"].shape[0], case["hq"], case["hkv"], d,
                                          s["tables"].shape[1], BLOCK, s["q"].dtype)  # fmt: skip
            s["ws"] = torch.empty(max(n, 256), dtype=torch.uint8, device="cuda")
        ops.paged_decode_fp8(s["out"], s["q"], *cache, s["tables"], s["ctx"], d**-0.5, s["ws"])
        return s["out"]
    ops.paged_prefill_fp8(s["out"], s["q"], *cache, s["tables"], s["qsl"], s["ctx"], s["qmax"],
                          d**-0.5)  # fmt: skip
    return s["out"]


def _store(s, k, v):
    """Writes float32 rows ``[T, Hkv, D]`` into the pools at the step's slots."""
    keep = s["slots"] >= 0
    slot = s["slots"][keep]
    blk, off = slot // BLOCK, slot % BLOCK
    for pool, scales, x in (("kp", "ks", k), ("vp", "vs", v)):
        x = x[keep]
        if s[scales] is None:
            s[pool][blk, :, off] = x.to(s[pool].dtype)
        else:
            sc = (x.abs().amax(-1) / E4M3_MAX).clamp_min(MIN_SCALE)
            q = (x / sc[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
            s[pool].view(torch.uint8)[blk, :, off] = q.view(torch.uint8)
            s[scales][blk, :, off] = sc
    return _written(s)


def _append(s):
    return _store(s, s["k"].float(), s["v"].float())


def _rotary(s):
    c = s["case"]
    t, d, rd, hq, hkv = s["qkv"].shape[0], c["d"], c["rd"], c["hq"], c["hkv"]
    x = s["qkv"].view(t, hq + 2 * hkv, d)
    # The angles in 64 bits: at position 1e5 a 32-bit product is off by more than 1e-3.
    ang = s["pos"].double()[:, None] * s["inv_freq"].double()[None, :]
    cos = (ang.cos() * s["mscale"]).float()[:, None, :]
    sin = (ang.sin() * s["mscale"]).float()[:, None, :]
    rot = x[:, : hq + hkv, :rd].float()
    if c["interleaved"]:
        a, b = rot[..., 0::2], rot[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = rot[..., : rd // 2], rot[..., rd // 2 :]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    qk = torch.cat((y, x[:, : hq + hkv, rd:].float()), -1)
    s["q_out"].copy_(qk[:, :hq].to(s["q_out"].dtype))
    return _store(s, qk[:, hq:], x[:, hq + hkv :].float())


def _values(pool, scales, index):
    """float32 values of cache rows at an index into (block, head[, offset])."""
    return pool.view(torch.uint8)[index].view(torch.float8_e4m3fn).float() * scales[index][..., None]


def _read(s):
    loc = s["loc"].long()
    t = s["k_out"].shape[0]
    row = torch.arange(t, device="cuda")
    seq = torch.searchsorted(loc, row, right=True) - 1
    pos = row - loc[seq]
    blk, off = s["tables"][seq, pos // BLOCK].long(), pos % BLOCK
    at = (blk[:, None], torch.arange(s["case"]["hkv"], device="cuda")[None, :], off[:, None])
    s["k_out"].copy_(_values(s["kp"], s["ks"], at).to(s["k_out"].dtype))
    s["v_out"].copy_(_values(s["vp"], s["vs"], at).to(s["v_out"].dtype))
    return s["k_out"], s["v_out"]


def _context(s, pool, scales):
    """Padded contexts ``[sequences, kv heads, width * BLOCK, dim]`` in float32."""
    tab = s["tables"].long()
    at = (tab[:, None, :], torch.arange(s["case"]["hkv"], device="cuda")[None, :, None])
    return _values(s[pool], s[scales], at).flatten(2, 3)


def _softmax(sc):
    """Rows that see nothing become zeros."""
    m = sc.amax(-1, keepdim=True).clamp_min(-1e30)
    p = sc.sub_(m).exp_()
    return p.div_(p.sum(-1, keepdim=True).clamp_min(1e-30))


def _decode(s):
    b, hq, d = s["q"].shape
    hkv = s["case"]["hkv"]
    q = s["q"].float().view(b, hkv, hq // hkv, d) * d**-0.5
    k = _context(s, "kp", "ks")
    sc = q @ k.transpose(-1, -2)
    del k
    hidden = torch.arange(sc.shape[-1], device="cuda")[None, :] >= s["ctx"][:, None]
    p = _softmax(sc.masked_fill_(hidden[:, None, None, :], -math.inf))
    v = _context(s, "vp", "vs")
    return (p @ v).view(b, hq, d).to(s["q"].dtype)


def _prefill(s):
    t, hq, d = s["q"].shape
    hkv = s["case"]["hkv"]
    qsl = s["qsl"].long()
    n = qsl[1:] - qsl[:-1]
    j = torch.arange(s["qmax"], device="cuda")
    real = j[None, :] < n[:, None]
    at = (qsl[:-1, None] + j[None, :]).clamp_max(t - 1)
    q = s["q"][at].float() * d**-0.5  # [sequences, qmax, heads, dim]
    q = q.unflatten(2, (hkv, hq // hkv)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    k = _context(s, "kp", "ks")
    sc = q @ k.transpose(-1, -2)
    del k
    pos = (s["ctx"].long() - n)[:, None] + j[None, :]
    hidden = torch.arange(sc.shape[-1], device="cuda")[None, None, :] > pos[:, :, None]
    sc = sc.unflatten(2, (hq // hkv, -1)).masked_fill_(hidden[:, None, None], -math.inf)
    p = _softmax(sc).flatten(2, 3)
    v = _context(s, "vp", "vs")
    o = (p @ v).unflatten(2, (hq // hkv, -1)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return o[real].to(s["q"].dtype)


# ------------------------------------------------------------------------------ 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    op, d, hkv = case["op"], case["d"], case["hkv"]
    if op == "append":
        return _exact_cache(s, s["k"].double(), s["v"].double())
    if op == "rotary":
        t, rd, hq = s["qkv"].shape[0], case["rd"], case["hq"]
        x = s["qkv"].double().view(t, hq + 2 * hkv, d)
        ang = torch.outer(s["pos"].double(), s["inv_freq"].double())
        # Pair (a + ib) times the factor and e^(i angle).
        turn = torch.polar(torch.full_like(ang, s["mscale"]), ang)[:, None, :]
        first = list(range(0, rd, 2)) if case["interleaved"] else list(range(rd // 2))
        second = [i + 1 for i in first] if case["interleaved"] else [i + rd // 2 for i in first]
        z = torch.complex(x[:, : hq + hkv, first], x[:, : hq + hkv, second]) * turn
        y = x.clone()
        y[:, : hq + hkv, first], y[:, : hq + hkv, second] = z.real, z.imag
        return _exact_cache(s, y[:, hq : hq + hkv], y[:, hq + hkv :]) | {"q_out": y[:, :hq]}
    if op == "read":
        return tuple(torch.cat([_exact_rows(s, p, sc, i, n) for i, n in enumerate(_lens(case))])
                     for p, sc in (("kp", "ks"), ("vp", "vs")))  # fmt: skip
    group = case["hq"] // hkv
    if op == "decode":
        lens, q_of, base = _lens(case), lambda i: s["q"][i : i + 1], None
    else:
        nq, np_ = _lens(case)
        lens, at = nq + np_, np.concatenate([[0], np.cumsum(nq)])
        q_of, base = lambda i: s["q"][at[i] : at[i + 1]], np_
    out = []
    for i, n in enumerate(lens.tolist()):
        q = q_of(i).double()
        if n == 0:
            out.append(torch.zeros_like(q))
            continue
        k = _exact_rows(s, "kp", "ks", i, n).repeat_interleave(group, 1)
        sc = torch.einsum("qhd,khd->hqk", q, k) / math.sqrt(d)
        del k
        if base is not None:
            see = torch.arange(n, device="cuda")[None, :] <= (
                int(base[i]) + torch.arange(q.shape[0], device="cuda")[:, None])  # fmt: skip
            sc = torch.where(see[None], sc, -math.inf)
        p = torch.softmax(sc, -1)
        v = _exact_rows(s, "vp", "vs", i, n).repeat_interleave(group, 1)
        out.append(torch.einsum("hqk,khd->qhd", p, v))
    return torch.cat(out)


def _exact_rows(s, pool, scales, i, n):
    """The first n rows of sequence i, ``[n, kv heads, dim]`` in 64 bits."""
    blk = s["tables"][i].long()
    x = s[pool].view(torch.uint8)[blk].view(torch.float8_e4m3fn).double()
    x = x * s[scales][blk].double().unsqueeze(-1)
    return x.transpose(1, 2).flatten(0, 1)[: int(n)]


def _exact_cache(s, k, v):
    """What the cache holds after a write, unrounded: x / scale, and the scales."""
    got = {}
    for pool, scales, x in (("kp", "ks", k), ("vp", "vs", v)):
        b, h, w, d = s[pool].shape
        held = torch.zeros(b * w, h, d, dtype=torch.float64, device="cuda")
        sc = torch.full((b * w, h), MIN_SCALE, dtype=torch.float64, device="cuda")
        live = torch.nonzero(s["slots"] >= 0).flatten()
        if s[scales] is None:
            held[s["slots"][live]] = x[live]
        else:
            sc[s["slots"][live]] = (x[live].abs().amax(-1) / 448).clamp_min(MIN_SCALE)
            held[s["slots"][live]] = x[live] / sc[s["slots"][live]].unsqueeze(-1)
            got[scales] = sc.view(b, w, h).transpose(1, 2).contiguous()
        got[pool] = held.view(b, w, h, d).transpose(1, 2).contiguous()
    return got
