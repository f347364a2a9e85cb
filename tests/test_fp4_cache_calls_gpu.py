"""A key-value cache in 4 bits on the device: calls that its documentation allows beside the usual ones."""
import math
import os
import pathlib
import subprocess
import sys

import pytest
import torch

from tests.fp4_oracle import attend, step
from tests.test_fp4_cache_calls import LAYOUTS
from tests.test_fp4_cache_calls import test_positions_outside_the_table as on_host
from tests.test_fp4_cache_gpu import _check as check
from tests.test_fp4_cache_gpu import _llm
from tests.test_fp4_cache_models import count_axes, image_prompts, logprobs
from vllm_b200 import ops
from vllm_b200.ops import cuda_ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H", [1, 2])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_keys_and_values_of_any_layout(layout, H):
    T, D, BS = 3, 16, 16
    with torch.device("cuda"):
        k, v = (LAYOUTS[layout](T, H, D) for _ in range(2))
    cache, want = (torch.zeros(ops.fp4_cache_shape(1, H, BS, D), dtype=torch.uint8, device=d) for d in ("cuda", "cpu"))
    slots = torch.tensor([5, 0, 9])
    ops.reshape_and_cache_fp4(k, v, cache, slots.cuda())
    ops.reshape_and_cache_fp4(k.cpu(), v.cpu(), want, slots)
    assert torch.equal(cache.cpu(), want)


@pytest.mark.parametrize("Hkv,G,D,few", [(64, 1, 128, 1100), (40, 1, 64, 1639), (32, 4, 192, 513)])
def test_many_heads_and_a_long_request_in_one_kernel(Hkv, G, D, few):
    """kv heads times query rows of a request beyond 16 bits, in the kernel of single tokens."""
    cu, Hq, BS, scale = cuda_ops(), Hkv * G, 32, D ** -0.5
    q, cache, md = step([40, 90], [3, 70], Hq, Hkv, D, BS, torch.bfloat16, "cuda", seed=D, spread=2.0)
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
    cu._fp4_few(q, cache, md, Hkv, D, BS, md.block_table.shape[1] * BS, scale, None, 0.0, out, lse, None, 1.0, few)
    want, norm, mass, terms, big = attend(q, cache, md, scale)
    # as for other steps: 32-bit sums of D products, a factor and an exponential; weights in fp16; 32-bit sums; the output's rounding
    eps = (D / 8 + 16) * 2.0 ** -23 * terms + 8 * 2.0 ** -24 * 1.5 * terms + 2.0 ** -21
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2 * eps + 2.0 ** -13) * mass + 90 * 2.0 ** -31 * big + 2.0 ** -25
    assert ((out.double().cpu() - want).abs() <= bound).all() and ((lse.double().cpu() - norm).abs() <= eps + 2.0 ** -20 + 2.0 ** -22 * norm.abs()).all()


def invariant_generation():
    from vllm_b200 import SamplingParams
    llm, r = _llm("llama-small", kv_cache_dtype="nvfp4", max_num_batched_tokens=64, enable_prefix_caching=False)
    assert cuda_ops().batch_invariant() and not r.graphs and not r.mixed_graphs
    sp = SamplingParams(max_tokens=8, temperature=0.0, ignore_eos=True, logprobs=0)
    prompts = [{"prompt_token_ids": [(7 * i + j) % 4000 + 3 for j in range(20 + 41 * i)]} for i in range(4)]

    def run(some):
        return [(o.outputs[0].token_ids, [x.logprob for d in o.outputs[0].logprobs for x in d.values()]) for o in llm.generate(some, sp)]

    together = run(prompts)
    assert [run([p])[0] for p in prompts] == together
    llm.shutdown()
    print("as alone")


def test_generation_in_batch_invariant_mode():
    """Runs without captured steps, and a request's tokens and log-probabilities are those that it has alone.  (A process of its own: the mode changes settings of the whole process.)"""
    got = subprocess.run([sys.executable, "-c", f"import {__name__} as t; t.invariant_generation()"], env={**os.environ, "VLLM_BATCH_INVARIANT": "1"}, capture_output=True, text=True,
                         timeout=300, cwd=pathlib.Path(__file__).parents[1])
    assert got.returncode == 0 and "as alone" in got.stdout, got.stdout[-2000:] + got.stderr[-2000:]


@pytest.mark.parametrize("queries", [[1], [40]])
@pytest.mark.parametrize("odd", [1001, 1004])
def test_queries_out_of_rows_of_any_width(queries, odd):
    """One token's queries in a row whose width is no multiple of 16 bytes: their distance to the next row counts as contiguous."""
    q, cache, md = step([300], queries, 6, 2, 64, 32, torch.bfloat16, "cuda", seed=9)
    want, norm = ops.paged_attention_fp4(q, cache, md, 0.125, return_lse=True)
    n = queries[0]
    wide = torch.zeros(n + 1, odd, dtype=q.dtype, device="cuda")
    wide[:n, :384] = q.flatten(1)
    one = wide[:, :384].unflatten(1, (6, 64))[:n]
    assert one.stride(0) == odd and one.is_contiguous() == (n == 1)
    got, lse = ops.paged_attention_fp4(one, cache, md, 0.125, return_lse=True)
    assert torch.equal(got, want) and torch.equal(lse, norm)
    out = torch.full_like(wide, 7.0)
    assert torch.equal(ops.paged_attention_fp4(one, cache, md, 0.125, out=out[:, :384].unflatten(1, (6, 64))[:n]), want) and (out[:, 384:] == 7.0).all() and (out[n] == 7.0).all()


def test_one_row_is_read_into_rows_of_any_width():
    """A row's distance to the next says nothing where there is one row; of more rows each has to lie at a 16-byte address."""
    H, D, BS = 2, 64, 32
    _, cache, md = step([300], [1], H, H, D, BS, torch.bfloat16, "cuda", seed=9)
    kv = torch.full((2, 2, 133), 7.0, dtype=torch.bfloat16, device="cuda")
    k, v = kv[0, :, :128].unflatten(1, (H, D)), torch.empty(2, H, D, dtype=torch.bfloat16, device="cuda")
    cu, first = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 1], [299]))
    ops.gather_cache_fp4(cache, md.block_table, cu, k[:1], v[:1], 1, first)
    want = [torch.empty(1, H, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    ops.gather_cache_fp4(cache, md.block_table, cu, *want, 1, first)
    assert torch.equal(k[:1], want[0]) and torch.equal(v[:1], want[1]) and (kv[0, 0, 128:] == 7.0).all() and (kv[0, 1] == 7.0).all()
    with pytest.raises(ValueError):
        ops.gather_cache_fp4(cache, md.block_table, cu, k, v, 1, first)
    _, cache, md = step([300], [1], 1, 1, D, BS, torch.bfloat16, "cuda", seed=9)
    heads_first = [torch.empty(1, 2, D, dtype=torch.bfloat16, device="cuda").transpose(0, 1) for _ in range(2)]              # one head
    want = [torch.empty(2, 1, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for got in (heads_first, want):
        ops.gather_cache_fp4(cache, md.block_table, torch.tensor([0, 2], dtype=torch.int32, device="cuda"), *got, 2)
    assert all(torch.equal(a, b) for a, b in zip(heads_first, want))


@pytest.mark.parametrize("D,Hq", [(128, 8), (192, 8), (48, 8)])
@pytest.mark.parametrize("padding", [0, 3])
def test_a_step_without_tokens(D, Hq, padding):
    """Requests wait, none has new tokens; ``max_query_len`` is a bound."""
    _, cache, md = step([40, 0], [0, 0], Hq, 2, D, 32, torch.bfloat16, "cuda")
    md.decode_only = False
    for md.max_query_len in (0, 1, 500):
        q = torch.full((padding, Hq, D), float("nan"), dtype=torch.bfloat16, device="cuda")
        got, lse = ops.paged_attention_fp4(q, cache, md, 1.0, return_lse=True)
        assert got.shape == q.shape and lse.shape == (padding, Hq) and (got == 0).all()
        out = torch.full_like(q, 7.0)
        assert ops.paged_attention_fp4(q, cache, md, 1.0, out=out) is out and (out == 7.0).all()


@pytest.mark.parametrize("axes", [False, True])
def test_positions_outside_the_table(axes):
    on_host(axes, "cuda", torch.bfloat16)


@pytest.mark.parametrize("model", ["gemma2-tiny", "gptoss-tiny", "qwen2vl-tiny", "qwen3moe-tiny", "bloom-tiny"])
def test_families_take_a_cache_in_4_bits(model):
    """Heads of 16 or 32, pages of 16: nothing to refuse."""
    llm, r = _llm(model, kv_cache_dtype="nvfp4", max_model_len=256, max_num_batched_tokens=64, block_size=16, kv_cache_memory_bytes=32 << 20)
    assert any(c.dtype == torch.uint8 for c in r.kv_caches.values())
    llm.shutdown()


@pytest.mark.parametrize("preset", ["qwen2vl-tiny", "qwen3vl-tiny", "qwen35vl-tiny"])
def test_an_image_turns_keys_by_three_axes(monkeypatch, preset):
    """Beside a text in a step, then single tokens; text alone in front of it gives the tokens that it has without the image."""
    from vllm_b200 import SamplingParams
    calls = count_axes(monkeypatch)
    llm, _ = _llm(preset, kv_cache_dtype="nvfp4", max_model_len=256, max_num_batched_tokens=64, block_size=16, kv_cache_memory_bytes=32 << 20, hf_overrides={"min_pixels": 32 * 32}, enable_prefix_caching=False)
    sp = SamplingParams(max_tokens=4, temperature=0.0, ignore_eos=True, logprobs=0)
    image, text = image_prompts()
    outs = llm.generate([image, text], sp)
    assert 3 in calls and all(len(x) == 4 and all(map(math.isfinite, x)) for x in logprobs(outs))
    calls.clear()
    alone = llm.generate([text], sp)
    assert 3 not in calls and max(abs(a - b) for a, b in zip(logprobs(alone)[0], logprobs(outs)[1])) < 0.05       # (some steps of bf16 in the logits, below 4)
    llm.shutdown()


def test_refused_offsets_name_the_call():
    q, cache, md = step([40, 90], [3, 70], 8, 2, 64, 32, torch.bfloat16, "cuda")
    good = md.query_start_loc
    for md.query_start_loc in (None, good.long(), good[:2], good.cpu(), good.repeat_interleave(2)[::2]):
        with pytest.raises(ValueError, match="paged_attention_fp4"):
            ops.paged_attention_fp4(q, cache, md, 1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("queries", [[1, 1, 1, 1], [3, 1, 40, 5]])
@pytest.mark.parametrize("Hq,Hkv,D,kw", [(4, 2, 128, {}), (6, 2, 64, {}), (4, 2, 192, {}), (4, 2, 48, {}), (3, 1, 160, {"window": 64}), (8, 2, 512, {"cap": 5.0}), (80, 1, 128, {}), (80, 1, 16, {}),
                                         (4, 2, 128, {"alibi_slopes": 1}), (4, 2, 96, {"alibi_slopes": 1}), (4, 2, 128, {"chunk_size": 32}), (6, 2, 64, {"chunk_size": 32}),
                                         (4, 2, 128, {"causal": False}), (4, 2, 80, {"causal": False}), (32, 2, 64, {"causal": False})])
def test_rows_without_keys(dtype, queries, Hq, Hkv, D, kw):
    """Requests with no rows in the cache, or fewer than new tokens: rows in front of the cache's first see no key (all of them where the mask is not causal), whatever was in memory."""
    if "alibi_slopes" in kw:
        kw = {"alibi_slopes": torch.linspace(0.01, 0.2, Hq).cuda()}
    for host in (True, False):
        for sinks in (None, torch.randn(Hq).cuda()):
            q, cache, md = step([0, 70, 33, 2], queries, Hq, Hkv, D, 32, dtype, "cuda", seed=D, spread=2.0, host=host)
            for x in [torch.full(q.shape, math.nan, dtype=dtype, device="cuda"), torch.full(q.shape[:2], math.nan, device="cuda")]:
                del x                        # (what an allocation without values finds next)
            got = check(q, cache, md, sinks=sinks, pages=True, **kw)
            assert (got[:queries[0]] == 0).all()


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16), (192, torch.bfloat16), (48, torch.bfloat16)])
@pytest.mark.parametrize("window", [1, 63, 64, 65, 700])
def test_windows_far_shorter_than_the_cache(D, dtype, window):
    q, cache, md = step([20000, 7001, 20000, 9000], [100, 30, 3, 1], 2, 1, D, 64, dtype, "cuda", seed=window, spread=2.0)
    check(q, cache, md, window=window, pages=True)


@pytest.mark.parametrize("queries", [[1, 1, 1], [5, 4, 5], [100, 1, 90]])
@pytest.mark.parametrize("D", [64, 128, 256, 48])
def test_the_same_call_gives_the_same_bits(D, queries):
    q, cache, md = step([3000, 90, 1000], queries, 8, 2, D, 32, torch.bfloat16, "cuda", seed=D, spread=2.0)
    first = ops.paged_attention_fp4(q, cache, md, D ** -0.5, return_lse=True)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(ops.paged_attention_fp4(q, cache, md, D ** -0.5, return_lse=True), first))


@pytest.mark.parametrize("D,Hq", [(64, 6), (128, 8), (192, 4), (48, 4)])
@pytest.mark.parametrize("path", ["rule", "straight", "pages", "few"])
def test_a_captured_step_of_prompts_follows_its_lengths(monkeypatch, D, Hq, path):
    """Without lengths on the host a step may be captured: replayed with other lengths and other new tokens of each request it gives what an eager call does."""
    if path != "rule":
        few = {"straight": 8, "pages": 8, "few": 200}[path]
        monkeypatch.setattr(cuda_ops(), "fp4_kernels", lambda T, B, longest, rows, H, G, D: (min(longest, few), path == "straight" or D > 128))
    q, cache, md = step([700, 300, 900], [150, 1, 40], Hq, 2, D, 32, torch.bfloat16, "cuda", seed=D, spread=2.0, host=False)
    md.max_query_len, md.max_seq_len = 200, 900
    other = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 10, 190, 191], [60, 300, 33])]
    ops.paged_attention_fp4(q, cache, md, 0.1)       # (what a first call sets up)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = ops.paged_attention_fp4(q, cache, md, 0.1, return_lse=True)
    for qsl, lens in ((md.query_start_loc.clone(), md.seq_lens.clone()), other):
        md.query_start_loc.copy_(qsl)
        md.seq_lens.copy_(lens)
        graph.replay()
        want, norm = ops.paged_attention_fp4(q, cache, md, 0.1, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, norm)
    check(q, cache, md, pages=True)


@pytest.mark.parametrize("Hq,Hkv,D,lens,queries", [(6, 2, 64, [3000, 500], [900, 40]), (8, 2, 128, [30000], [700]), (4, 2, 256, [9000], [100]), (4, 2, 48, [4000, 4000], [1, 30]), (40, 1, 64, [900] * 30, [5] * 30),
                                                   (5, 1, 96, [2000] * 9, [90] * 9)])
@pytest.mark.parametrize("host", [True, False])
def test_memory_of_a_step(monkeypatch, Hq, Hkv, D, lens, queries, host):
    """What a call takes beside its outputs is within what the engine keeps free, whichever kernels it goes to."""
    cu = cuda_ops()
    q, cache, md = step(lens, queries, Hq, Hkv, D, 64, torch.bfloat16, "cuda", host=host)
    for path in ("rule", "straight", "pages"):
        if path != "rule":
            monkeypatch.setattr(cu, "fp4_kernels", lambda T, B, longest, rows, H, G, D: (min(longest, 4), path == "straight" or D > 128))
        for most in (1 << 30, 1 << 22):
            monkeypatch.setattr(cu, "FP4_PAGES_BYTES", most)
            out = torch.empty_like(q)
            ops.paged_attention_fp4(q, cache, md, 0.1, out=out)
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            ops.paged_attention_fp4(q, cache, md, 0.1, out=out)
            torch.cuda.synchronize()
            # (beside 512 bytes for each allocation)
            assert torch.cuda.max_memory_allocated() - before <= cu.fp4_step_bytes(q.shape[0], len(lens), max(lens), Hq, Hkv, D) + (1 << 16)


CAPTURED_FIRST = """
import torch
from tests.fp4_oracle import step
from vllm_b200 import ops
runs = []
for D, lens, queries in ((128, [70, 2000], [1, 1]), (64, [300] * 200, [1] * 200), (64, [400, 90], [5, 2]), (192, [700, 90], [300, 1]), (128, [700, 90], [300, 1]), (48, [70, 90], [1, 1])):
    q, cache, md = step(lens, queries, 8, 2, D, 32, torch.bfloat16, "cuda", host=False)
    runs.append((q, cache, md, D))
k = torch.randn(6, 2, 64, device="cuda").bfloat16()
to, slots, table = torch.zeros(ops.fp4_cache_shape(1, 2, 16, 64), dtype=torch.uint8, device="cuda"), torch.arange(6, device="cuda"), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
cu = torch.tensor([0, 6], dtype=torch.int32, device="cuda")

def run():
    out = [x for q, cache, md, D in runs for x in ops.paged_attention_fp4(q, cache, md, 0.1, return_lse=True)]
    ops.reshape_and_cache_fp4(k, -k, to, slots)
    back = [torch.empty_like(k) for _ in range(2)]
    ops.gather_cache_fp4(to, table, cu, *back, 6)
    return out + back

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run()
graph.replay()
torch.cuda.synchronize()
got = [x.clone() for x in got]
assert all(torch.equal(a, b) for a, b in zip(got, run()))
"""


def test_first_calls_in_a_capture():
    """Before anything has run on the device."""
    r = subprocess.run([sys.executable, "-c", CAPTURED_FIRST], capture_output=True, text=True, timeout=300, cwd=pathlib.Path(__file__).parents[1])
    assert r.returncode == 0, r.stderr[-2000:]
