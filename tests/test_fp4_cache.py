"""A key-value cache in 4 bits: plain operations against the definition, refusals, rules of dispatch, and generation with one (CPU)."""
import math
import types

import pytest
import torch

from tests.fp4_oracle import CODES, SCALES, attend, quantise, step, values
from tests.utils import llama_full_weights, make_llm
from vllm_b200 import SamplingParams, ops
from vllm_b200.config.model import get_preset_hf_config
from vllm_b200.ops import cuda, ref


def _cache(blocks=4, H=2, BS=16, D=32):
    return torch.zeros(ops.fp4_cache_shape(blocks, H, BS, D), dtype=torch.uint8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scales", [(1.0, 1.0), (0.75, 1.3)])
def test_written_and_read_rows_are_the_definition(dtype, scales):
    H, D, BS, T = 2, 48, 16, 7
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(T, H, D, generator=g) * torch.logspace(-3, 2, T)[:, None, None] for _ in range(2))
    k[2, 0, :16], k[3, 0, 3], k[4, 1, 20] = 0.0, math.nan, math.inf
    k, v = k.to(dtype), v.to(dtype)
    slots = torch.tensor([5, 40, -1, 17, 63, 64, 0])            # one nowhere, one behind the cache
    cache = _cache(4, H, BS, D)
    ops.reshape_and_cache_fp4(k, v, cache, slots, *scales)
    got = values(cache)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < 64:
            for part, x in enumerate((k, v)):
                for h in range(H):
                    codes, e = quantise(x[t, h].tolist(), scales[part])
                    want = CODES[torch.tensor(codes)] * SCALES[torch.tensor(e)].repeat_interleave(16)
                    assert torch.equal(got[s // BS, part, h, s % BS].nan_to_num(1e9), want.nan_to_num(1e9))
    untouched = [s for s in range(64) if s not in slots.tolist()]
    assert all((got[s // BS, :, :, s % BS] == 0).all() for s in untouched)
    kk, vv = (torch.empty(3, H, D, dtype=torch.float32) for _ in range(2))
    ops.gather_cache_fp4(cache, torch.tensor([[2, 1]], dtype=torch.int32), torch.tensor([0, 3], dtype=torch.int32), kk, vv, 3, torch.tensor([30], dtype=torch.int32), *scales)
    f = torch.tensor(scales, dtype=torch.float32)
    assert torch.equal(kk[:2].double(), (got[1, 0, :, 14:].transpose(0, 1).float() * f[0]).double()) and (kk[2] == 0).all() and (vv[2] == 0).all()


def test_a_row_stands_within_half_a_step_of_its_values():
    """Codes are at most half a step (1 of 6 at the top, of a scale off by at most 2^-4) from the values."""
    x = torch.randn(64, 1, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    cache = _cache(4, 1, 16, 128)
    ops.reshape_and_cache_fp4(x, x, cache, torch.arange(64))
    y = values(cache)[:, 0].transpose(1, 2).reshape(64, 1, 128)
    top = x.double().unflatten(-1, (8, 16)).abs().amax(-1, keepdim=True)
    err = (x.double() - y).unflatten(-1, (8, 16)).abs() / top
    assert err.max() <= (1 + 2.0 ** -4) / 6 + 2.0 ** -4 and err.mean() < 0.05


@pytest.mark.parametrize("kw", [{}, {"window": 7, "cap": 20.0, "factors": (0.5, 2.0)}])
def test_attention_is_that_of_the_values(kw):
    q, cache, md = step([5, 40, 33], [1, 3, 33], 4, 2, 32, 16, torch.float32, "cpu", seed=3, spread=2.0)
    sinks = torch.randn(4) if kw else None
    want, norm, mass, _, _ = attend(q, cache, md, 0.2, sinks=sinks, **kw)
    factors = kw.get("factors", (1.0, 1.0))
    got, lse = ops.paged_attention_fp4(q, cache, md, 0.2, kw.get("window"), kw.get("cap", 0.0), sinks=sinks, return_lse=True, k_scale=factors[0], v_scale=factors[1])
    assert ((got.double() - want).abs() <= 1e-5 * mass + 1e-6).all() and (lse.double() - norm).abs().max() < 1e-4


@pytest.mark.parametrize("neox", [True, False])
def test_rotation_on_several_axes(neox):
    T, Hq, H, D, rot, far = 5, 4, 2, 32, 16, 50
    g = torch.Generator().manual_seed(4)
    q, k, v = torch.randn(T, Hq * D, generator=g), torch.randn(T, H * D, generator=g), torch.randn(T, H * D, generator=g)
    table = torch.randn(far, rot, generator=g)
    positions = torch.randint(0, far, (3, T), generator=g)
    axes = torch.tensor([0, 1, 2, 2, 1, 0, 0, 1], dtype=torch.int32)
    own = torch.cat([torch.stack([table[positions[axes[j]], half * rot // 2 + j] for j in range(rot // 2)], 1) for half in range(2)], 1)     # a row for each token
    want_q, want_k = ref.rotary_embedding(torch.arange(T), q.clone(), k.clone(), own, D, neox)
    cache, plain, k0 = _cache(), _cache(), k.clone()
    got = ops.rope_and_cache_fp4(positions, q, k, v, table, D, neox, cache, torch.arange(T), axes=axes)
    ops.reshape_and_cache_fp4(want_k.view(T, H, D), v.view(T, H, D), plain, torch.arange(T))
    assert got is q and torch.equal(q, want_q.view_as(q)) and torch.equal(cache, plain) and torch.equal(k, k0)


def test_refusals():
    cache, x, s = _cache(), torch.zeros(3, 2, 32), torch.zeros(3, dtype=torch.int64)
    for bad in ((16, 8), (16, 40), (8, 32), (24, 32)):
        with pytest.raises(ValueError):
            ops.fp4_cache_shape(4, 2, *bad)
    for k, v, c, slots, scale in ((x, x, cache.char(), s, 1.0), (x, x, cache[..., :17], s, 1.0), (x, x, cache.transpose(0, 1), s, 1.0), (x, x[:2], cache, s, 1.0), (x, x.half(), cache, s, 1.0),
                                  (x[:, :1], x[:, :1], cache, s, 1.0), (x, x, cache, s[:2], 1.0), (x, x, cache, s.int(), 1.0), (x, x, cache, s, 0.0), (x, x, cache, s, math.nan)):
        with pytest.raises(ValueError):
            ops.reshape_and_cache_fp4(k, v, c, slots, scale)
    q, k, table, pos = torch.zeros(3, 128), torch.zeros(3, 64), torch.zeros(9, 32), torch.zeros(3, dtype=torch.int64)
    for args, kw in (((pos, q, k, k, table, 64, True, cache, s), {}), ((pos, q[:, :100], k, k, table, 32, True, cache, s), {}), ((pos, q, k[:2], k, table, 32, True, cache, s), {}),
                     ((pos.int(), q, k, k, table, 32, True, cache, s), {}), ((pos, q, k, k, table.double(), 32, True, cache, s), {}),
                     ((pos, q, k, k, torch.zeros(9, 34), 32, True, cache, s), {}), ((pos, q, k, k, table, 32, True, cache, s), {"axes": torch.zeros(16, dtype=torch.int32)}),
                     ((pos[None], q, k, k, table, 32, True, cache, s), {"axes": torch.zeros(15, dtype=torch.int32)}),
                     ((pos[None], q, k, k, table, 32, True, cache, s), {"axes": torch.zeros(16)})):
        with pytest.raises(ValueError):
            ops.rope_and_cache_fp4(*args, **kw)
    cu, bt = torch.tensor([0, 3], dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    for c, t, n, a, b in ((cache, bt.long(), cu, x, x), (cache, bt, cu.long(), x, x), (cache, bt[:0], cu, x, x), (cache, bt, cu, x, x.half()), (cache, bt, cu, x[:, :1], x), (cache[0], bt, cu, x, x)):
        with pytest.raises(ValueError):
            ops.gather_cache_fp4(c, t, n, a, b, 3)
    q, cache, md = step([5, 9], [1, 1], 4, 2, 32, 16, torch.float32, "cpu")
    for kw in ({"sinks": torch.zeros(3)}, {"alibi_slopes": torch.zeros(5)}, {"out": torch.empty(2, 4, 16)}, {"out": torch.empty(2, 4, 32, dtype=torch.float16)}, {"v_scale": -1.0}):
        with pytest.raises(ValueError):
            ops.paged_attention_fp4(q, cache, md, 1.0, **kw)
    for bad in (q[:, :3], q[:, :, :16], q[:1]):
        with pytest.raises(ValueError):
            ops.paged_attention_fp4(bad, cache, md, 1.0)
    md.kv_vt = True
    with pytest.raises(ValueError):
        ops.paged_attention_fp4(q, cache, md, 1.0)


def test_runs_of_requests_fit_into_the_workspace(monkeypatch):
    """All requests with more than a few new tokens, in order, each once, and no run above the limit unless it is one request."""
    monkeypatch.setattr(cuda, "FP4_PAGES_BYTES", 1000)
    import numpy as np
    rng = np.random.default_rng(0)
    for trial in range(50):
        B = int(rng.integers(1, 9))
        queries, lens = rng.integers(0, 12, B), rng.integers(0, 400, B)
        md = types.SimpleNamespace(num_reqs=B, decode_only=False, seq_lens_cpu=None, host_lens=(np.concatenate(([0], queries.cumsum())), lens) if trial % 2 else None)
        runs = cuda._fp4_runs(md, 4, 64, 7, 100)
        assert [r[0] for r in runs] == [0, *[r[1] for r in runs[:-1]]] and runs[-1][1] == B
        for first, end, total, longest in runs:
            need = [(0 if queries[b] <= 4 else max(1, min(7, -(-int(lens[b]) // 64)))) if trial % 2 else 7 for b in range(first, end)]
            assert total == sum(need) and longest == max(need) and (total * 100 <= 1000 or sum(n > 0 for n in need) == 1)


def test_every_request_has_one_kernel():
    """New tokens up to which the kernel of single tokens is taken: at least the base, never more than the longest."""
    for T, B, longest, rows, H, G, D in ((64, 64, 1, 1000, 8, 4, 128), (80, 16, 5, 4000, 8, 4, 128), (8000, 1, 8000, 8000, 8, 4, 128), (1000, 2, 500, 12000, 4, 4, 64), (3, 1, 3, 3, 1, 64, 256),
                                         (500, 1, 500, 500, 1, 1, 192)):
        few, straight = cuda.fp4_kernels(T, B, longest, rows, H, G, D)
        assert min(longest, max(1, 64 // G)) <= few <= longest and few * G <= 4096 and (straight or D <= 128)


def _runner(llm):
    return llm.llm_engine.engine_core.engine_core.model_executor.worker.runner


def test_generation_with_a_cache_in_4_bits():
    cfg = get_preset_hf_config("llama-tiny")
    w = list(llama_full_weights(cfg, seed=3))
    sp = SamplingParams(max_tokens=2, temperature=0.0, ignore_eos=True, prompt_logprobs=0)
    p = [{"prompt_token_ids": [(5 * i) % 400 + 3 for i in range(40)]}]
    res, blocks = {}, {}
    for kvd in ("auto", "nvfp4"):
        llm = make_llm("llama-tiny", weights=w, kv_cache_dtype=kvd, max_num_batched_tokens=16)   # chunked: reads the cache
        o = llm.generate(p, sp)[0]
        res[kvd] = [list(d.values())[0].logprob for d in o.prompt_logprobs[1:]]
        r = _runner(llm)
        blocks[kvd] = r.kv_cache_config.num_blocks
        if kvd == "nvfp4":
            cache, layer = next(iter(r.kv_caches.values())), r.model
            assert cache.dtype == torch.uint8 and cache.shape[1:] == ops.fp4_cache_shape(1, cache.shape[2], cache.shape[3], cache.shape[4] * 16 // 9)[1:] and layer is not None
        llm.shutdown()
    assert 0 < max(abs(a - b) for a, b in zip(res["auto"], res["nvfp4"])) < 0.5
    assert blocks["nvfp4"] >= 7 * blocks["auto"] - 7                                             # 9 / 16 of a byte for 4 (models of 32 bits here)


@pytest.mark.parametrize("preset", ["qwen2vl-tiny", "gemma2-tiny", "gptoss-tiny", "bloom-tiny", "jamba-tiny", "qwen3moe-tiny"])
def test_families_run_with_a_cache_in_4_bits(preset):
    cfg = get_preset_hf_config(preset)
    try:
        llm = make_llm(preset, kv_cache_dtype="nvfp4", load_format="dummy", block_size=16)
    except ValueError as e:
        assert "4 bits" in str(e) and cfg is not None          # heads that are no multiple of 16
        return
    out = llm.generate([{"prompt_token_ids": [5, 7, 11, 13] * 6}], SamplingParams(max_tokens=4, temperature=0.0, ignore_eos=True))
    assert len(out[0].outputs[0].token_ids) == 4
    llm.shutdown()


@pytest.mark.parametrize("preset", ["pomipel-tiny", "kopadra-tiny", "gizilorn-tiny", "legelix-tiny"])
def test_layers_that_write_their_own_caches_refuse(preset):
    with pytest.raises(ValueError, match="nvfp4|fp8|4 bits"):
        make_llm(preset, kv_cache_dtype="nvfp4", load_format="dummy")


def test_pages_that_are_no_multiple_of_16_refuse():
    with pytest.raises(ValueError, match="nvfp4"):
        make_llm("llama-tiny", kv_cache_dtype="nvfp4", load_format="dummy", block_size=8)


def test_the_choice_of_kernel_looks_at_prompts_alone(monkeypatch):
    """Single tokens beside a prompt, whatever their number and their lengths, do not move the choice for it where lengths are on the host."""
    monkeypatch.setattr(cuda, "fp4_kernels", lambda T, B, longest, rows, H, G, D: (longest, (T, B, longest, rows)))

    def asked(queries, lens, room, host=True):
        cu = [sum(queries[:i]) for i in range(len(lens) + 1)]
        md = types.SimpleNamespace(num_reqs=len(lens), max_seq_len=max(lens), host_lens=(cu, lens) if host else None)
        return cuda._fp4_choice(md, max(queries), 4, cu[-1], room, 2, 128)

    assert asked([400], [700], 1 << 20) == (400, (400, 1, 400, 700))
    assert asked([1, 400, 1, 1], [90000, 700, 5, 800], 1 << 20) == (16, (400, 1, 400, 700))
    assert asked([100, 300], [4000, 400], 1 << 20) == (300, (400, 2, 300, 1300)) and asked([100, 300], [4000, 400], 1000)[1][3] == 1000
    assert asked([100, 300], [4000, 400], 5000, host=False) == (300, (400, 2, 300, 4000)) and asked([3, 2], [4000, 9], 5000) == (3, (5, 2, 3, 4000))


def test_range_of_prompts():
    import numpy as np
    for new, few, want in (([1, 1, 40, 2, 90, 1], 4, (2, 3)), ([5], 4, (0, 1)), ([4, 4], 4, (0, 0)), ([], 0, (0, 0)), ([0, 0, 1], 0, (2, 1)), ([9, 1], 1, (0, 1))):
        assert cuda._fp4_range(np.array(new, dtype=np.int64), few) == want
