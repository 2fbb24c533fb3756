"""What the 8-bit cache operators refuse, on the host and before any launch (CPU only)."""

from __future__ import annotations

import pytest
import torch

from tokenserve_b200 import _build, ops

BF = torch.bfloat16


@pytest.fixture(scope="module")
def lib():  # type: ignore[no-untyped-def]
    _build.build()
    return ops.load_library()


def cache(nb=4, h=2, bs=16, d=64):  # type: ignore[no-untyped-def]
    p = torch.zeros(nb, h, bs, d, dtype=torch.uint8).view(torch.float8_e4m3fn)
    return p, p.clone(), torch.ones(nb, h, bs), torch.ones(nb, h, bs)


def test_c_entry_points_check_their_arguments(lib) -> None:  # type: ignore[no-untyped-def]
    one = 0x1000  # never read: every call below is refused first

    def append(dtype=ops.TS_BFLOAT16, t=4, h=8, d=128, bs=16, ks=one, stride=1024, key=one, tags=None):
        return lib.ts_reshape_and_cache_fp8(key, one, stride, stride, one, one, ks, one, one, t, h, d,
                                            bs, 10, dtype, tags, None, None, None)  # fmt: skip

    assert append(dtype=7) == -1 and b"bad dtype" in lib.ts_last_error()
    assert append(d=0) == -1 and b"bad sizes" in lib.ts_last_error()
    assert append(t=-1) == -1
    assert append(ks=None) == -1 and b"null pointer" in lib.ts_last_error()
    assert append(stride=1023) == -1 and b"stride" in lib.ts_last_error()
    assert append(tags=one) == -1 and b"go together" in lib.ts_last_error()
    assert append(key=one + 1) == -4 and append(ks=one + 2) == -4
    assert append(t=0) == 0 and lib.ts_last_error() == b""

    def rotary(dtype=ops.TS_BFLOAT16, t=4, hq=32, rd=128, ks=one, vs=one, stride=6144, q=one, pos=one):
        return lib.ts_rotary_and_cache(one, stride, q, one, one, ks, vs, one, pos, one, t, hq, 8, 128,
                                       rd, 0, 1.0, 16, 10, dtype, None, None)  # fmt: skip

    assert rotary(dtype=3) == -1 and b"bad dtype" in lib.ts_last_error()
    assert rotary(hq=0) == -1 and b"bad sizes" in lib.ts_last_error()
    for rd in (0, 129, 130, 63, -2):
        assert rotary(rd=rd) == -1 and b"rotary_dim" in lib.ts_last_error()
    assert rotary(stride=6143) == -1 and b"stride" in lib.ts_last_error()
    assert rotary(vs=None) == -1 and b"go together" in lib.ts_last_error()
    assert rotary(pos=None) == -1 and b"null pointer" in lib.ts_last_error()
    assert rotary(q=one + 1) == -4
    assert rotary(t=0) == 0

    def read(dtype=ops.TS_BFLOAT16, seqs=2, t=10, width=4, loc=one, out=one):
        return lib.ts_read_cache_fp8(out, one, one, one, one, one, one, width, loc, seqs, t, 8, 128,
                                     16, 10, dtype, None, None)  # fmt: skip

    assert read(dtype=-1) == -1 and read(width=0) == -1 and read(t=-1) == -1
    assert read(loc=None) == -1 and b"null pointer" in lib.ts_last_error()
    assert read(out=one + 1) == -4
    assert read(t=0) == 0 and read(seqs=0) == 0

    def decode(dtype=ops.TS_BFLOAT16, b=2, hq=32, ks=one, stride=4096, q=one, ws=None, wsn=0, nb=10):
        return lib.ts_paged_decode_fp8(one, q, stride, one, one, ks, one, one, 8, one, b, hq, 8, 128,
                                       16, nb, 0.1, dtype, ws, wsn, 0, None)  # fmt: skip

    assert decode(dtype=9) == -1 and decode(hq=30) == -1 and decode(b=-1) == -1
    assert decode(ks=None) == -1 and b"scales" in lib.ts_last_error()
    assert decode(ks=one + 1) == -4
    assert decode(q=None) == -1 and decode(stride=4095) == -1
    assert decode(b=0, ks=None) == 0

    def prefill(dtype=ops.TS_BFLOAT16, seqs=2, t=8, qmax=4, hq=32, stride=4096, vs=one, out=one):
        return lib.ts_paged_prefill_fp8(out, one, stride, one, one, one, vs, one, 8, one, one, seqs,
                                        t, qmax, hq, 8, 128, 16, 10, 0.1, dtype, None)  # fmt: skip

    assert prefill(dtype=5) == -1 and prefill(hq=33) == -1 and prefill(qmax=-1) == -1
    assert prefill(stride=100) == -1 and prefill(vs=None) == -1
    assert prefill(out=one + 1) == -4 and prefill(vs=one + 2) == -4
    assert prefill(seqs=0) == 0 and prefill(t=0) == 0 and prefill(qmax=0) == 0


def refused(fn, *args, match, **kw):  # type: ignore[no-untyped-def]
    with pytest.raises(ops.KernelError, match=match):
        fn(*args, **kw)


def test_wrappers_refuse_other_pools_and_host_tensors(lib) -> None:  # type: ignore[no-untyped-def]
    kp, vp, ks, vs = cache()
    x, slots = torch.zeros(3, 2, 64, dtype=BF), torch.zeros(3, dtype=torch.int64)
    f = ops.reshape_and_cache_fp8
    refused(f, x, x, kp.view(torch.uint8), vp, ks, vs, slots, match="float8_e4m3fn")
    refused(f, x, x, kp, vp[:3], ks, vs, slots, match="float8_e4m3fn")
    refused(f, x, x, kp[:, :, :, :32], vp[:, :, :, :32], ks, vs, slots, match="contiguous")
    refused(f, x, x, kp, vp, ks.double(), vs, slots, match="scales")
    refused(f, x, x, kp, vp, ks, vs[:, :1], slots, match="scales")
    refused(f, x, x, kp, vp, ks, vs, slots, match="CUDA device")
    tab, ctx = torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    q = torch.zeros(3, 4, 64, dtype=BF)
    refused(ops.paged_decode_fp8, q.clone(), q, kp, vp, ks, vs, tab, ctx, 0.1, None,
            match="CUDA device")  # fmt: skip
    refused(ops.paged_decode_fp8, q.clone(), q, kp.view(torch.uint8), vp, ks, vs, tab, ctx, 0.1, None,
            match="float8_e4m3fn")  # fmt: skip
    refused(ops.paged_prefill_fp8, q.clone(), q, kp, vp, ks, vs, tab, torch.zeros(4), ctx, 1, 0.1,
            match="CUDA device")  # fmt: skip
    refused(ops.read_cache_fp8, x, x, kp, vp, ks, vs, tab, ctx, match="CUDA device")
    qkv = torch.zeros(3, 8 * 64, dtype=BF)
    refused(ops.rotary_and_cache, qkv, q, kp, vp, slots, slots, torch.ones(32), 4, 2, key_scales=ks,
            match="go together")  # fmt: skip
    refused(ops.rotary_and_cache, qkv, q, kp, vp, slots, slots, torch.ones(32), 4, 2,
            match="qkv's dtype")  # fmt: skip


def test_backend_config_refuses_unknown_caches_and_shards() -> None:
    from tokenserve_b200.backend import CudaPagedBackendConfig

    assert CudaPagedBackendConfig(kv_cache_dtype="fp8_e4m3").kv_cache_dtype == "fp8_e4m3"
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        CudaPagedBackendConfig(kv_cache_dtype="int8")
    with pytest.raises(ValueError, match="kv_head_shards"):
        CudaPagedBackendConfig(kv_cache_dtype="fp8_e4m3", kv_head_shards=2)
