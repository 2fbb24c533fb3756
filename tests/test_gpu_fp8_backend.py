"""CudaPagedBackend with an 8-bit KV cache (GPU): what the cache holds, graphs against eager steps,
block copy and swap, scaled rotary positions, shadow-KV checks, refusals."""

from __future__ import annotations

import asyncio

import pytest
import torch

from tests.fp8_reference import rows_of
from tokenserve_b200.backend import CudaPagedBackend, CudaPagedBackendConfig
from tokenserve_b200.interface import BatchItem

pytestmark = pytest.mark.gpu

VOCAB = 97


def llama(dtype=torch.float32, **over):  # type: ignore[no-untyped-def]
    import transformers

    cfg = dict(vocab_size=VOCAB, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
               num_attention_heads=4, num_key_value_heads=2, head_dim=64, rope_theta=10000.0,
               max_position_embeddings=2048, attn_implementation="eager")  # fmt: skip
    cfg.update(over)
    torch.manual_seed(3)
    return transformers.LlamaForCausalLM(transformers.LlamaConfig(**cfg)).to(dtype).eval()


def backend(model, **over):  # type: ignore[no-untyped-def]
    cfg = dict(block_size=16, num_blocks=64, device="cuda:0", kv_cache_dtype="fp8_e4m3")
    cfg.update(over)
    return CudaPagedBackend(model, CudaPagedBackendConfig(**cfg))


def item(seq, tokens, start, table):  # type: ignore[no-untyped-def]
    return BatchItem(seq_id=seq, token_ids=list(tokens), start=start,
                     num_new_tokens=len(tokens) - start, num_prompt_tokens=len(tokens),
                     block_table=list(table), sample=True, seed=0)  # fmt: skip


def run(b, batch):  # type: ignore[no-untyped-def]
    return asyncio.run(b.execute(batch))


PROMPTS = {1: [(i * 7) % VOCAB for i in range(40)], 2: [(i * 5 + 1) % VOCAB for i in range(9)]}
TABLES = {1: [5, 3, 9, 20], 2: [7, 12]}


def generate(b, steps, tables=TABLES, toks=None, hook=None):  # type: ignore[no-untyped-def]
    """Greedy tokens of both sequences; ``hook(step)`` may move them to other tables."""
    if toks is None:
        toks = {s: list(p) for s, p in PROMPTS.items()}
        got = run(b, [item(s, toks[s], 0, tables[s]) for s in toks])
        for s, t in got.items():
            toks[s].append(t)
    for step in range(steps):
        if hook is not None:
            tables = hook(step) or tables
        got = run(b, [item(s, toks[s], len(toks[s]) - 1, tables[s]) for s in toks])
        for s, t in got.items():
            toks[s].append(t)
    return toks


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_graph_replay_equals_eager_steps(cuda_device, dtype) -> None:  # type: ignore[no-untyped-def]
    model = llama(dtype)
    eager = backend(model, cuda_graphs=False)
    want = generate(eager, 6)
    graphs = backend(model, cuda_graphs=True)
    assert graphs.runner.fused and generate(graphs, 6) == want
    # Both prompts ran as the same eager step. (Rows of decode steps may differ in fp32 sums: a graph
    # pads the batch to 8 rows, and the projections' GEMMs of another height add in another order.)
    assert bool((eager.read_kv(TABLES[1], 40) == graphs.read_kv(TABLES[1], 40)).all())


def test_cache_holds_the_quantised_rows_of_the_first_layer(cuda_device) -> None:  # type: ignore[no-untyped-def]
    """Layer 0 projects the embeddings, which the cache does not touch, so its K and V rows are those
    of a float32 cache: each value is at most half an e4m3 step off (2^-4 of it, or 2^-10 of the
    row's scale), plus what separates the two fp32 rotations: the plain path takes the angle's
    product in fp32, off by 2^-24 of at most 40 radians, and rounds each product."""
    model = llama()
    plain, quant = backend(model, kv_cache_dtype=None), backend(model)
    for b in (plain, quant):
        generate(b, 0)
    for s, table in TABLES.items():
        n = len(PROMPTS[s])
        x, y = plain.read_kv(table, n)[0].double(), quant.read_kv(table, n)[0].double()
        amax = x.abs().amax(-1, keepdim=True)
        lim = torch.maximum(x.abs() * 2.0**-4, amax / 448 * 2.0**-10) + amax * 2 * 40 * 2.0**-23
        assert ((x - y).abs() <= lim).all()
        assert quant.runner.cache(0)[0].dtype == torch.float8_e4m3fn
    assert quant.runner.block_bytes * 4 < plain.runner.block_bytes * 1.1  # 64 + 4 of 256 bytes a row


def test_modules_path_and_shadow_verification(cuda_device) -> None:  # type: ignore[no-untyped-def]
    """With verify_kv the transformers modules run and K/V go through reshape_and_cache_fp8: the cache
    agrees with the fused path's to one e4m3 step (values fp32 rounding apart that round to
    neighbouring codes) and the scales to 40 2^-22, the rotations' fp32 differences (see above)."""
    model = llama()
    fused, modules = backend(model), backend(model, verify_kv=True)
    for b in (fused, modules):
        generate(b, 0)
    for a, c in zip(fused.runner.cache(0), modules.runner.cache(0), strict=True):
        if a.dtype == torch.float32:
            assert ((a - c).abs() <= c.abs() * 40 * 2.0**-22).all()
        else:
            # e4m3 codes order like their magnitudes as bytes; the sign bit apart.
            u, v = a.view(torch.uint8).int(), c.view(torch.uint8).int()
            mag = ((u & 127) - (v & 127)).abs()
            same_sign = (u & 128) == (v & 128)
            assert ((mag <= 1) & (same_sign | ((u & 127) + (v & 127) <= 1))).all()
            assert float((u != v).double().mean()) < 0.01


@pytest.mark.parametrize("rope", [
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
     "original_max_position_embeddings": 64, "rope_theta": 10000.0},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64,
     "rope_theta": 10000.0},
    {"rope_type": "linear", "factor": 2.0, "rope_theta": 10000.0},
])  # fmt: skip
def test_scaled_rotary_positions_run_fused(cuda_device, rope) -> None:  # type: ignore[no-untyped-def]
    model = llama(rope_parameters=rope, max_position_embeddings=512)
    b = backend(model)
    assert b.runner.fused
    generate(b, 0)
    layer, rot = model.model.layers[0], model.model.rotary_emb
    with torch.no_grad():
        ids = torch.tensor(PROMPTS[1], device=cuda_device)
        x = layer.input_layernorm(model.model.embed_tokens(ids))
        k = layer.self_attn.k_proj(x).view(len(ids), 2, 64).double()
    ang = torch.outer(torch.arange(len(ids), device=cuda_device).double(), rot.inv_freq.double())
    c = (ang.cos() * rot.attention_scaling)[:, None]
    s = (ang.sin() * rot.attention_scaling)[:, None]
    want = torch.cat((k[..., :32] * c - k[..., 32:] * s, k[..., 32:] * c + k[..., :32] * s), -1)
    code, scale = rows_of(b.runner.cache(0)[0], b.runner.cache(0)[2],
                          torch.tensor(TABLES[1], device=cuda_device), len(ids))  # fmt: skip
    got = (code * scale[..., None]).transpose(0, 1)
    # Half an e4m3 step; the projections of the two runs may differ in their fp32 sums of 256
    # products (2^-24 each of at most amax, 256 of them).
    amax = want.abs().amax(-1, keepdim=True)
    lim = torch.maximum(want.abs() * 2.0**-4, amax / 448 * 2.0**-10) + amax * 2.0**-14
    assert ((got - want).abs() <= lim).all()


def test_dynamic_rotary_runs_through_the_modules(cuda_device) -> None:  # type: ignore[no-untyped-def]
    model = llama(rope_parameters={"rope_type": "dynamic", "factor": 2.0, "rope_theta": 10000.0})
    b = backend(model)
    assert not b.runner.fused
    assert len(generate(b, 2)[1]) == len(PROMPTS[1]) + 3


def test_copy_and_swap_carry_codes_and_scales(cuda_device) -> None:  # type: ignore[no-untyped-def]
    model = llama(torch.bfloat16)
    want = generate(backend(model), 6)
    b = backend(model, swap_space_blocks=8)
    toks = generate(b, 2)
    before = {s: b.read_kv(t, len(toks[s]) - 1) for s, t in TABLES.items()}
    b.copy_blocks([(5, 30), (3, 31), (9, 32), (20, 33)])
    b.swap_out([(7, 0), (12, 4)])
    b.runner.kv.view(torch.uint8)[:, :, [5, 3, 9, 20, 7, 12]] = 0x7F
    b.runner.kv_scales[:, :, [5, 3, 9, 20, 7, 12]] = float("nan")
    b.swap_in([(0, 40), (4, 41)])
    moved = {1: [30, 31, 32, 33], 2: [40, 41]}
    for s, t in moved.items():
        assert torch.equal(b.read_kv(t, len(toks[s]) - 1), before[s])
    for s in moved:
        b.free(s)  # the sequences come back with other tables, as after a preemption
    assert generate(b, 4, tables=moved, toks=toks) == want


def test_resize_and_read_kv_bounds(cuda_device) -> None:  # type: ignore[no-untyped-def]
    b = backend(llama())
    b.resize_pool(32)
    assert b.runner.kv.shape[2] == 32 and b.runner.kv_scales.shape[2] == 32
    assert b.runner.pool_bytes == 32 * b.runner.block_bytes
    assert b.read_kv([1, 2], 0).shape == (2, 2, 0, 2, 64)
    assert (b.read_kv([1, 2], 20) == 0).all()
    for table, n in (([1], 17), ([1, 32], 20), ([-1], 3), ([1], -1)):
        with pytest.raises(ValueError, match="read_kv"):
            b.read_kv(table, n)


def test_read_kv_of_a_plain_cache(cuda_device) -> None:  # type: ignore[no-untyped-def]
    b = backend(llama(torch.bfloat16), kv_cache_dtype=None)
    generate(b, 1)
    got = b.read_kv(TABLES[1], 41)
    kv = b.runner.kv
    for p in (0, 15, 16, 40):
        assert torch.equal(got[:, :, p], kv[:, :, TABLES[1][p // 16], :, p % 16])
