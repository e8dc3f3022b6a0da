"""An engine with an 8-bit key/value cache under speculation, preemption and later turns: rows that are written and taken back, blocks
that change hands, drafting heads with a layer of their own."""
import dataclasses

import pytest
import torch

from legion_b200 import ops
from legion_b200.config import tiny_gqa_moe
from legion_b200.engine.lm import EngineConfig, build_engine
from legion_b200.engine.types import GenerateRequest, SamplingParams
from legion_b200.models.weights import random_weights
from test_kv8_engine import CFGS, gpu, prompt

MODELS = {**CFGS, "mtp": lambda: dataclasses.replace(tiny_gqa_moe(), mtp_layers=1)}


def engine(name, device="cpu", **kw):
    cfg = MODELS[name]()
    base = dict(ctx_size=512, max_seqs=4, block_size=16, prefill_chunk=64, max_batch_tokens=128, kv_dtype="fp8", device=device)
    base.update(kw)
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    return build_engine(cfg, weights=random_weights(cfg, device, dtype, seed=0, std=0.05), engine_cfg=EngineConfig(**base))


def reply(eng, toks, n=20):
    return eng.generate_text(tokens=toks, max_tokens=n, ignore_eos=True).token_ids


@pytest.mark.parametrize("name,spec", [("dense", "ngram"), ("hybrid", "draft"), ("gqa_moe", "suffix"), ("gqa_moe", "draft"), ("gqa_moe", "eagle3"),
                                       ("mtp", "mtp"), ("mtp", "mtp_ngram"), ("dense", "dflash")])
def test_speculation_over_an_8_bit_cache(name, spec):
    """Verify steps write rows that are taken back; drafting heads keep an 8-bit layer of their own."""
    prompts = [prompt(60, 1), prompt(20, 1) * 4]
    plain, eng = engine(name, prefix_cache=False), engine(name, prefix_cache=False, spec=spec, spec_k=3)
    want, got = ([reply(e, p) for p in prompts] for e in (plain, eng))
    st = eng.stats()
    plain.shutdown()
    eng.shutdown()
    assert got == want and st.spec_verify_steps > 0


def test_preempted_sequences_are_recomputed():
    seeds = (1, 2, 3)
    eng = engine("gqa_moe", prefix_cache=False, kv_admission="on-demand", kv_cache_tokens=15 * 16, kv_swap_gib=1.0)
    streams = [eng.generate(GenerateRequest(prompt_tokens=prompt(100, s), sampling=SamplingParams(max_tokens=24, ignore_eos=True))) for s in seeds]
    got, st = [s.collect().token_ids for s in streams], eng.stats()
    eng.shutdown()
    want = []
    for s in seeds:
        e = engine("gqa_moe", prefix_cache=False)
        want.append(reply(e, prompt(100, s), 24))
        e.shutdown()
    assert got == want and st.kv_preemptions >= 1 and st.kv_swap_out == 0


def test_second_turn_goes_on_in_a_partly_filled_block():
    eng, cold = engine("hybrid"), engine("hybrid", prefix_cache=False)
    first = prompt(70, 4)
    a = reply(eng, first, 13)
    turn = first + a[:-1] + prompt(20, 5)
    b = eng.generate_text(tokens=turn, max_tokens=8, ignore_eos=True)
    want = reply(cold, turn, 8)
    eng.shutdown()
    cold.shutdown()
    assert b.token_ids == want and b.usage.cached_tokens == 82


@gpu
@pytest.mark.parametrize("name,spec", [("dense", "eagle3"), ("mtp", "mtp"), ("gqa_moe", "draft")])
def test_speculation_and_captured_steps(name, spec):
    """Drafts, verify steps and captured steps of one engine over the same 8-bit blocks: nothing is refused, and every reply ends."""
    device = "cuda:0"
    eng = engine(name, device, block_size=64, spec=spec, spec_k=3)
    rep = prompt(20, 1) * 4
    got = [reply(eng, p) for p in (prompt(70, 1), rep, rep)]
    st = eng.stats()
    eng.shutdown()
    assert [len(g) for g in got] == [20] * 3 and st.spec_verify_steps > 0
    torch.cuda.synchronize()
    assert ops.sm100.Workspace.get(device).check() == 0


@gpu
def test_blocks_written_on_the_gpu():
    """Layer 0 sees the same inputs with either cache, also across portions and decode steps: its blocks hold the codes of the rows that
    the 16-bit cache holds, encoded as the steps came."""
    device, toks, held = "cuda:0", prompt(150, 2), []
    for kind in ("auto", "fp8"):
        eng = engine("dense", device, kv_dtype=kind, prefix_cache=False, block_size=64)
        eng.generate_text(tokens=toks, max_tokens=1, ignore_eos=True)
        held.append((eng.kv.k[0], eng.kv.v[0]))
        eng.shutdown()
    (k, v), (c, _) = held
    used = [i for i in range(k.shape[0]) if bool(k[i].any())]
    assert len(used) == 3
    for plain, codes, scale in ((k, c.k, c.k_scale), (v, c.v, c.v_scale)):
        for i in used:
            x = plain[i].transpose(0, 1).float().cpu()
            s = scale[i].cpu()
            assert torch.equal(s, ops.reference.kv8_scale_of(x.abs().amax((1, 2))))
            got = codes[i].cpu().float() * s[:, None, None]
            assert bool(((got - x).abs() <= x.abs() * 2.0 ** -4 + s[:, None, None] * 2.0 ** -10).all())
