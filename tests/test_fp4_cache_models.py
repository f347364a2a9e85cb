"""A key-value cache in 4 bits in the engine: positions on several axes, families that have to take it."""
import pytest
import torch

from tests.utils import make_llm
from vllm_b200 import SamplingParams, ops


def _runner(llm):
    return llm.llm_engine.engine_core.engine_core.model_executor.worker.runner


def image_prompts():
    """An image with text around it, and text alone."""
    import numpy as np
    from PIL import Image
    img = Image.fromarray(np.random.default_rng(0).integers(0, 255, (56, 84, 3), dtype=np.uint8))
    return [{"prompt_token_ids": [5, 17, 99, 502, 500, 503, 3, 250, 41, 7], "multi_modal_data": {"image": img}}, {"prompt_token_ids": [5, 17, 99, 3, 250, 41]}]


def count_axes(monkeypatch):
    """Numbers of position axes of the calls to the rotating write, in order."""
    calls, write = [], ops.rope_and_cache_fp4

    def counted(positions, *args, axes=None, **kw):
        calls.append(1 if axes is None else positions.shape[0])
        return write(positions, *args, axes=axes, **kw)

    monkeypatch.setattr(ops, "rope_and_cache_fp4", counted)
    return calls


def logprobs(outs):
    return [[x.logprob for d in (o.prompt_logprobs or [])[1:] + o.outputs[0].logprobs for x in d.values()] for o in outs]


def seed_weights(model):
    g = torch.Generator().manual_seed(1)
    with torch.no_grad():
        for p in model.parameters():
            p.copy_((torch.randn(p.shape, generator=g) * 0.2 + (p.dim() == 1)).to(p.dtype))


@pytest.mark.parametrize("preset", ["qwen2vl-tiny", "qwen3vl-tiny", "qwen35vl-tiny"])
def test_an_image_turns_keys_by_three_axes(monkeypatch, preset):
    """An image's step takes the write with several axes (sections one after the other, interleaved, and of half a head).  Where a cache of the model's type is given
    the values that the other one stands for, both give the same log-probabilities, up to the order of 32-bit sums (some hundred terms of up to 2^-24 of a few units)."""
    sp = SamplingParams(max_tokens=4, temperature=0.0, ignore_eos=True, logprobs=0)
    write, got = ops.reshape_and_cache, {}

    def rounded(key, value, *args, **kw):
        return write(*(ops.ref.fp4_rows(*ops.ref.fp4_quant_rows(x)).to(x.dtype) for x in (key, value)), *args, **kw)

    for kvd in ("auto", "nvfp4"):
        if kvd == "nvfp4":
            calls = count_axes(monkeypatch)
        else:
            monkeypatch.setattr(ops, "reshape_and_cache", rounded)
            monkeypatch.setattr(ops, "rope_and_cache", lambda *args, vt=False: _turned(*args, rounded))
        llm = make_llm(preset, kv_cache_dtype=kvd, load_format="dummy", block_size=16, enable_prefix_caching=False, hf_overrides={"min_pixels": 32 * 32})
        seed_weights(_runner(llm).model)
        outs = llm.generate(image_prompts(), sp)
        got[kvd] = [o.outputs[0].token_ids for o in outs], logprobs(outs)
        llm.shutdown()
        monkeypatch.undo()
    assert 3 in calls and 1 in calls
    assert got["auto"][0] == got["nvfp4"][0]
    assert max(abs(a - b) for x, y in zip(got["auto"][1], got["nvfp4"][1]) for a, b in zip(x, y)) < 2e-4


def _turned(positions, q, k, v, table, D, neox, cache, slots, write):
    q, k = ops.ref.rotary_embedding(positions, q, k, table, D, neox)
    write(k.reshape(k.shape[0], -1, D), v.reshape(v.shape[0], -1, D), cache, slots)
    return q, k


@pytest.mark.parametrize("preset", ["qwen2vl-tiny", "gemma2-tiny", "gptoss-tiny", "bloom-tiny", "jamba-tiny", "qwen3moe-tiny"])
def test_families_take_a_cache_in_4_bits(preset):
    """Heads of 16 or 32, pages of 16: nothing to refuse."""
    llm = make_llm(preset, kv_cache_dtype="nvfp4", load_format="dummy", block_size=16)
    assert any(c.dtype == torch.uint8 for c in _runner(llm).kv_caches.values())
    llm.shutdown()
