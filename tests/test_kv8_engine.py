"""The engine with an 8-bit key/value cache: what its layers read and write, batches, portions of prompts, prefix reuse, captured
decode steps with padded rows, refusals."""
import pytest
import torch

from legion_b200 import ops
from legion_b200.config import tiny_dense, tiny_gqa_moe, tiny_hybrid_moe, tiny_mla_moe, tiny_muse
from legion_b200.engine.lm import EngineConfig, build_engine
from legion_b200.engine.types import GenerateRequest, SamplingParams
from legion_b200.models.decoder import KvCache
from legion_b200.models.weights import random_weights

gpu = pytest.mark.gpu
CFGS = {"hybrid": tiny_hybrid_moe, "gqa_moe": tiny_gqa_moe, "dense": tiny_dense, "window": tiny_muse}


def prompt(n, seed=1, vocab=255):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def engine(name, device="cpu", **kw):
    cfg = CFGS[name]()
    base = dict(ctx_size=512, max_seqs=4, block_size=16, prefill_chunk=64, max_batch_tokens=128, kv_dtype="fp8", device=device)
    base.update(kw)
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    return build_engine(cfg, weights=random_weights(cfg, device, dtype, seed=0, std=0.05), engine_cfg=EngineConfig(**base))


def alone(name, seeds, device="cpu", n=12, **kw):
    out = []
    for s in seeds:
        eng = engine(name, device, prefix_cache=False, **kw)
        out.append(eng.generate_text(tokens=prompt(70 + 9 * s, s), max_tokens=n, ignore_eos=True).token_ids)
        eng.shutdown()
    return out


def together(name, seeds, device="cpu", n=12, **kw):
    eng = engine(name, device, **kw)
    streams = [eng.generate(GenerateRequest(prompt_tokens=prompt(70 + 9 * s, s), sampling=SamplingParams(max_tokens=n, ignore_eos=True)))
               for s in seeds]
    got = [s.collect().token_ids for s in streams]
    eng.shutdown()
    return got


@pytest.mark.parametrize("name", list(CFGS))
def test_batched_equals_single(name):
    assert together(name, (1, 2, 3), prefix_cache=False) == alone(name, (1, 2, 3))


def test_prefix_reuse_equals_recomputing():
    eng = engine("dense")
    toks = prompt(120, 4)
    got = [eng.generate_text(tokens=toks, max_tokens=8, ignore_eos=True).token_ids for _ in range(2)]
    eng.shutdown()
    assert got[0] == got[1]


def test_the_cache_holds_the_encoded_keys_and_values():
    """Layer 0 sees the same inputs with either cache: its blocks hold what ``kv8_append`` makes of them."""
    toks = prompt(50, 2)
    held = []
    for kind in ("auto", "fp8"):
        eng = engine("dense", kv_dtype=kind, prefix_cache=False)
        eng.generate_text(tokens=toks, max_tokens=1, ignore_eos=True)
        held.append((eng.kv.k[0], eng.kv.v[0]))
        eng.shutdown()
    (k, v), (c, c2) = held
    assert c is c2 and isinstance(c, ops.Kv8Cache)
    used = [i for i in range(k.shape[0]) if bool(k[i].any())]
    got_used = [i for i in range(c.k.shape[0]) if bool(c.k_scale[i].any())]
    assert used == got_used and len(used) == 4
    for plain, codes, scale in ((k, c.k, c.k_scale), (v, c.v, c.v_scale)):
        values = codes.float() * scale[..., None, None]
        for i in used:
            x = plain[i].transpose(0, 1)                               # [heads, page, dim]
            assert torch.equal(scale[i], ops.reference.kv8_scale_of(x.abs().amax((1, 2))))
            # half a step of e4m3: 2^-4 of the value, 2^-10 of the scale below the smallest normal one
            assert bool(((values[i] - x).abs() <= x.abs() * 2.0 ** -4 + scale[i][:, None, None] * 2.0 ** -10).all())


def test_half_the_bytes():
    cfg = tiny_dense()
    full, small = (KvCache(cfg, 2, 64, "cpu", torch.bfloat16, kv8=q).bytes_per_block() for q in (False, True))
    assert full / 2 < small <= full / 2 + cfg.n_layer * cfg.n_kv_head * 8


def test_copy_blocks():
    cache = KvCache(tiny_dense(), 4, 16, "cpu", torch.float32, kv8=True)
    c = cache.k[1]
    c.k.view(torch.uint8)[2], c.k_scale[2], c.v_scale[2] = 7, 0.5, 0.25
    cache.copy_blocks([2], [3])
    assert bool((c.k.view(torch.uint8)[3] == 7).all()) and float(c.k_scale[3, 0]) == 0.5 and float(c.v_scale[3, 0]) == 0.25


def test_refusals():
    with pytest.raises(ValueError, match="8-bit"):
        KvCache(tiny_mla_moe(), 4, 16, "cpu", torch.float32, kv8=True)
    with pytest.raises(ValueError, match="8-bit"):
        KvCache(tiny_dense(), 4, 128, "cpu", torch.float32, kv8=True)
    with pytest.raises(ValueError, match="kv_dtype"):
        engine("dense", kv_dtype="int3")
    with pytest.raises(ValueError, match="rings"):
        engine("window", kv_rings=True)


@gpu
@pytest.mark.parametrize("name", ["dense", "hybrid", "window"])
def test_captured_steps_with_padded_rows(name):
    """Three sequences in a bucket of four, eager and captured: the padded row writes nothing, not to block 0 either."""
    device = "cuda:0"
    runs = [together(name, (1, 2, 3), device, block_size=64, cuda_graphs=g, prefix_cache=False) for g in (False, True)]
    assert runs[0] == runs[1]
    torch.cuda.synchronize()
    assert ops.sm100.Workspace.get(device).check() == 0


@gpu
def test_batched_equals_single_captured():
    device = "cuda:0"
    assert together("gqa_moe", (1, 2), device, block_size=64, prefix_cache=False) == alone("gqa_moe", (1, 2), device, block_size=64)
    assert ops.sm100.Workspace.get(device).check() == 0
