"""A key-value cache with a budget on the device: values, shapes and calls at the edge of what the operators take."""
import dataclasses
import os
import subprocess
import sys

import pytest
import torch

from tests.key_budget_oracle import attend, step, unit, weight_error
from tests.test_key_budget_gpu import _check_decode, _check_weights
from vllm_b200 import ops
from vllm_b200.ops import cuda_ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,BS,vt", [(128, 64, True), (64, 16, False)])
def test_weights_capped_rows_that_differ(D, BS, vt):
    """Capped scores, log-sum-exps that change from tile to tile: each tile has its own, in every run the same bits."""
    q, cache, md, scores = step([2300], [2300], 8, 2, D, BS, torch.bfloat16, "cuda", vt=vt, seed=5)
    lse = 4 + 6 * torch.rand(2300, 8, generator=torch.Generator().manual_seed(2)).cuda()
    want = None
    for _ in range(10):
        got = scores.clone()
        _check_weights(q, cache, md, got, cap=30.0, lse=lse)
        assert want is None or torch.equal(got, want)
        want = got


@pytest.mark.parametrize("invariant", [False, True])
def test_refusals_in_front_of_attention(invariant, monkeypatch):
    """Prompts, and decode steps in batch-invariant mode: what the attention kernels would follow blindly is refused on the host."""
    if invariant:
        monkeypatch.setenv("VLLM_BATCH_INVARIANT", "1")
    replace = dataclasses.replace
    q, cache, md, scores = step([33, 5], [1, 1] if invariant else [20, 5], 8, 2, 128, 64, torch.bfloat16, "cuda", vt=True)
    many = [step([33, 5], [1, 1] if invariant else [20, 5], heads, 1, 128, 64, torch.bfloat16, "cuda", vt=vt) for heads, vt in ((5, True), (40, True), (129, False))]
    before = scores.clone()
    for q_, cache_, md_, scores_ in [(q, cache, replace(md, **change), scores) for change in (
            dict(block_table=md.block_table.cpu()), dict(block_table=md.block_table.long()), dict(block_table=md.block_table[:1]), dict(seq_lens=md.seq_lens.cpu()),
            dict(seq_lens=md.seq_lens[:1]), dict(query_start_loc=md.query_start_loc.cpu()), dict(query_start_loc=md.query_start_loc.long()),
            dict(query_start_loc=md.query_start_loc[:2]), dict(block_table=md.block_table[:, :0]))] + many:
        with pytest.raises(ValueError):
            ops.scored_attention(q_, cache_, md_, 0.1, scores_)
    with pytest.raises(ValueError):
        ops.scored_attention(q, cache, md, 0.0, scores)
    torch.cuda.synchronize()
    assert torch.equal(scores, before)


@pytest.mark.parametrize("invariant", [False, True])
@pytest.mark.parametrize("where", ["", "given", "odd", "wide"])
@pytest.mark.parametrize("D,BS,vt", [(128, 64, True), (64, 16, False), (80, 16, False)])
def test_padded_and_unaligned(invariant, where, D, BS, vt, monkeypatch):
    """Padding rows behind the last request, queries and outputs at odd addresses: the bits of a plain call, zeros (or what was there) behind them."""
    if invariant:
        monkeypatch.setenv("VLLM_BATCH_INVARIANT", "1")
    q, cache, md, scores = step([33, 70], [1, 1] if invariant else [20, 45], 8, 2, D, BS, torch.bfloat16, "cuda", vt=vt)
    used, other = q.shape[0], scores.clone()
    want = ops.scored_attention(q, cache, md, 0.1, other)
    q = torch.cat([q, torch.full_like(q[:1], float("nan")).expand(3, -1, -1)])
    T = q.shape[0]
    wide = torch.zeros(T, 8 * D + 5, dtype=q.dtype, device="cuda")
    wide[:, 5:] = q.flatten(1)
    q = wide[:, 5:].unflatten(1, (8, D))
    out = {"": None, "given": torch.full((T, 8, D), 7.0, dtype=q.dtype, device="cuda"), "odd": torch.full((T * 8 * D + 4,), 7.0, dtype=q.dtype, device="cuda")[4:].view(T, 8, D),
           "wide": torch.full((T, 8 * D + 5), 7.0, dtype=q.dtype, device="cuda")[:, 5:].unflatten(1, (8, D))}[where]
    got = ops.scored_attention(q, cache, md, 0.1, scores, out=out)
    assert torch.equal(got[:used], want) and torch.equal(scores, other) and (got[used:] == (0.0 if out is None else 7.0)).all()
    assert out is None or got is out


def _check_sums(q, cache, md, scores, scale, lse, cap=0.0, last=0):
    """``_check_weights`` for scales of either sign, with log-sum-exps that may be larger than the scores: the factor, the product, the parts and the
    sums that they join (at most D / 16 + 4 additions, cut or rounded) are off by 2^-23 of them each."""
    D, turn = q.shape[2], -1 if scale < 0 else 1
    given = torch.where(lse.isfinite(), lse, torch.inf)
    _, _, weights, _, terms = attend(q * turn, cache, md, scale * turn, cap, None, last, given)
    size = float(lse[lse.isfinite()].abs().max())
    before = scores.clone()
    ops.key_weights(q, cache, md, scale, lse, scores, cap, last)
    n = weights.shape[2]
    total = before.double()
    total[:, :, :n] += weights
    bound = 2.0 ** -24 * total
    bound[:, :, :n] += (weight_error(terms, D) + (D / 16 + 4) * 2.0 ** -23 * size + 38 * 2.0 ** -24) * weights + 2.0 ** -126
    assert ((scores.double() - total).abs() <= bound).all(), ((scores.double() - total).abs() / bound.clamp(min=1e-300)).max()
    seen = torch.arange(scores.shape[2], device="cuda") < md.seq_lens[:, None, None]
    assert torch.equal(scores[~seen.expand_as(scores)], before[~seen.expand_as(scores)])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,D,BS,vt", [(8, 2, 128, 64, True), (9, 1, 64, 16, False), (6, 2, 256, 32, False)])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_weights_infinite(dtype, Hq, Hkv, D, BS, vt, cap):
    """Rows whose log-sum-exp is infinite or NaN give nothing, in tiles that all rows see and in those on the diagonal."""
    q, cache, md, scores = step([900, 400], [300, 400], Hq, Hkv, D, BS, dtype, "cuda", vt=vt, seed=1)
    lse = attend(q, cache, md, D ** -0.5, cap)[1].float()
    lse[::3], lse[1::5], lse[2::7] = float("inf"), float("-inf"), float("nan")
    _check_sums(q, cache, md, scores, D ** -0.5, lse, cap)
    lse[:, 1:] = float("inf")
    _check_sums(q, cache, md, scores, D ** -0.5, lse, cap)


@pytest.mark.parametrize("Hq,Hkv,D,BS,vt", [(8, 2, 128, 64, True), (9, 1, 64, 16, False), (33, 1, 128, 32, False), (10, 2, 256, 16, False)])
@pytest.mark.parametrize("scale,cap", [(-0.1, 0.0), (-0.1, 30.0), (0.1, 0.0), (0.1, 30.0)])
def test_weights_of_either_sign(Hq, Hkv, D, BS, vt, scale, cap):
    """Scales below 0, also where heads x tokens of a tile leave columns that nothing uses."""
    q, cache, md, scores = step([900, 200], [300, 200], Hq, Hkv, D, BS, torch.bfloat16, "cuda", vt=vt, seed=2)
    turn = -1 if scale < 0 else 1
    lse = attend(q * turn, cache, md, scale * turn, cap)[1].float()
    _check_sums(q, cache, md, scores, scale, lse, cap)


@pytest.mark.parametrize("dtype,scale,spread", [(torch.float16, 1e-7, 1.0), (torch.float16, 1e-10, 1.0), (torch.float16, 64.0, 2.0 ** -7), (torch.float16, -64.0, 2.0 ** -7),
                                                (torch.bfloat16, 1e-10, 1.0), (torch.bfloat16, 3e-38, 1.0), (torch.bfloat16, 1e-40, 1.0), (torch.bfloat16, 64.0, 2.0 ** -7)])
@pytest.mark.parametrize("D,BS", [(8, 16), (128, 32)])
def test_weights_of_small_and_large_scales(dtype, scale, spread, D, BS):
    """Scales whose quotients with the log-sum-exps do not fit into the cache's type, or are small in it."""
    q, cache, md, scores = step([700, 90], [200, 90], 4, 2, D, BS, dtype, "cuda", seed=3, spread=spread)
    turn = -1 if scale < 0 else 1
    _check_sums(q, cache, md, scores, scale, attend(q * turn, cache, md, scale * turn)[1].float())


def _small_numbers(q, cache):
    """Queries and keys of -1, 0 and 1 (in place): their products are exact in any order."""
    q.copy_(q.round().clamp(-1, 1))
    keys = cache[:, 0]
    keys.copy_(keys.nan_to_num(0.0).round().clamp(-1, 1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,D,BS,vt", [(4, 128, 64, True), (5, 64, 16, False), (2, 256, 32, False)])
@pytest.mark.parametrize("cap", [5.0, 30.0, 50.0])
@pytest.mark.parametrize("scale", [1 / 64, 1 / 4, 4.0])
def test_weights_capped_exactly(dtype, H, D, BS, vt, cap, scale):
    """Weights of one query row and head each, its products exact: what is left is the error of the cap and of the exponential."""
    q, cache, md, scores = step([2000, 300], [300, 300], H, H, D, BS, dtype, "cuda", vt=vt, seed=6)
    _small_numbers(q, cache)
    scores.zero_()
    lse = torch.zeros(600, H, device="cuda") if scale < 0.1 else attend(q, cache, md, scale, cap)[1].float()
    ops.key_weights(q, cache, md, scale, lse, scores, cap, last=1)
    want = attend(q, cache, md, scale, cap, None, 1, lse)[2]
    for b, n in enumerate([2000, 300]):
        last = lse[300 * b + 299].double()[:, None]
        size = (want[b, :, :n].log() + last).abs()                             # of the capped scores
        # the cap: its factors, two products and a polynomial of 1.6e-7 (or an exponential of 2^-22 below 1 / 4 of it, a reciprocal and a
        # difference); the log-sum-exp: a factor and a product; the difference of both; an exponential of 2^-22; two sums
        error = size * (5 * 2.0 ** -24 + 1.6e-7) + last.abs() * 2.0 ** -23 + (size + last.abs()) * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -23
        off = (scores[b, :, :n].double() - want[b, :, :n]).abs() / want[b, :, :n]
        assert (off <= error + 2.0 ** -126 / want[b, :, :n]).all(), (off / error).max()


def _check_prompt(q, cache, md, scores, scale, cap=0.0, sinks=None, last=0, out=None):
    """Output and scores of a prompt whose queries and keys are small whole numbers (``_small_numbers``), against 64 bits."""
    D, n_max = q.shape[2], max(md.seq_lens.tolist())
    want, norm, weights, mass, terms = attend(q, cache, md, scale, cap, sinks, last)
    before = scores.clone()
    got = ops.scored_attention(q, cache, md, scale, scores, logits_soft_cap=cap, sinks=sinks, last=last, out=out)
    assert out is None or got is out
    lse = float(norm[norm.isfinite()].abs().max())
    size = min(terms, cap or terms)                                            # of the scores, whose products are exact
    # a weight of the attention: factors and differences of its exponent, the cap (5 roundings and 1.6e-7), an exponential; the log-sum-exp: chains of 64
    # weights in a tile, of the tiles and of warps (up to 130 additions), a logarithm, its factors
    weight = 6 * 2.0 ** -24 * (size + lse) + (5 * 2.0 ** -24 + 1.6e-7) * size * (cap > 0) + 2.0 ** -22
    of_lse = weight + 130 * 2.0 ** -24 + 2.0 ** -22 * (lse + 1)
    # of a key: the same exponent, or the log-sum-exp in the middle of a product whose sums are cut (D / 32 + 3 of them left); chains of additions
    of_key = weight + of_lse + (D / 32 + 3) * 2.0 ** -23 * (terms + lse) * (cap == 0) + 38 * 2.0 ** -24
    u, n = unit(q.dtype), weights.shape[2]
    bound = u * want.abs() + (u + weight + of_lse + 2.0 ** -13) * mass + (2.0 ** -25 * (1 + 6 * n_max) if q.dtype is torch.float16 else 0.0)
    assert ((got.double() - want).abs() <= bound).all(), ((got.double() - want).abs() / bound).max()
    total = before.double()
    total[:, :, :n] += weights
    bound = 2.0 ** -24 * total
    bound[:, :, :n] += of_key * weights + 2.0 ** -126
    assert ((scores.double() - total).abs() <= bound).all(), ((scores.double() - total).abs() / bound.clamp(min=1e-300)).max()
    seen = torch.arange(scores.shape[2], device="cuda") < md.seq_lens[:, None, None]
    assert torch.equal(scores[~seen.expand_as(scores)], before[~seen.expand_as(scores)])


PROMPTS = [(8, 2, 128, 64, True), (16, 1, 128, 64, True), (3, 3, 128, 64, True), (8, 2, 64, 16, False), (24, 3, 64, 32, False), (10, 2, 64, 16, False), (8, 2, 96, 48, False),
           (6, 6, 80, 16, False), (8, 4, 128, 32, False), (4, 2, 256, 32, False), (33, 1, 128, 16, False), (2, 1, 8, 16, False)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,D,BS,vt", PROMPTS)
@pytest.mark.parametrize("cap,sink,last", [(0.0, False, 0), (0.0, True, 7), (30.0, False, 7), (4.0, True, 0)])
@pytest.mark.parametrize("where", ["", "strided"])
def test_prompts(dtype, Hq, Hkv, D, BS, vt, cap, sink, last, where):
    """Prompts through every kind of attention kernel: the log-sum-exps that they hand on hold the cap and the sinks."""
    lens, queries = [300, 1, 700, 0, 64, 130, 513], [300, 1, 45, 0, 1, 129, 3]
    q, cache, md, scores = step(lens, queries, Hq, Hkv, D, BS, dtype, "cuda", vt=vt, seed=Hq + D)
    _small_numbers(q, cache)
    out = None
    if where:
        T = q.shape[0]
        wide = torch.zeros(T, Hq * D + 24, dtype=dtype, device="cuda")
        wide[:, 16:-8] = q.flatten(1)
        q, out = wide[:, 16:-8].unflatten(1, (Hq, D)), torch.zeros(T, Hq + 3, D, dtype=dtype, device="cuda")[:, 2:-1]
    sinks = torch.randn(Hq, generator=torch.Generator().manual_seed(1)).cuda() if sink else None
    _check_prompt(q, cache, md, scores, D ** -0.5, cap, sinks, last, out)


@pytest.mark.parametrize("lens,queries,last", [([3000], [3000], 0), ([2500, 700], [2500, 700], 64), ([9000, 300], [20, 300], 0), ([40] * 130, [40] * 130, 0)])
@pytest.mark.parametrize("D,BS,vt", [(128, 64, True), (64, 16, False)])
def test_prompts_lengths(lens, queries, last, D, BS, vt):
    q, cache, md, scores = step(lens, queries, 8, 2, D, BS, torch.bfloat16, "cuda", vt=vt, seed=len(lens))
    _small_numbers(q, cache)
    _check_prompt(q, cache, md, scores, D ** -0.5, last=last)


@pytest.mark.parametrize("B,Hq,Hkv,rows", [(64, 32, 8, 131072), (300, 8, 1, 131072), (2, 256, 1, 600000)])
def test_decode_memory(B, Hq, Hkv, rows):
    """Buffers for far longer texts than there are: what a call allocates has a bound."""
    lens = [5 + 11 * i % 900 for i in range(B)]
    q, cache, md, scores = step(lens, [1] * B, Hq, Hkv, 128, 64, torch.bfloat16, "cuda", vt=True, seed=7)
    n = scores.shape[2]
    scores = torch.nn.functional.pad(scores, (0, rows - n))
    md.block_table = torch.nn.functional.pad(md.block_table, (0, rows // 64 - md.block_table.shape[1]))
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before, was = scores[:, :, :n].clone(), torch.cuda.memory_allocated()
    out = ops.scored_attention(q, cache, md, 0.1, scores)
    torch.cuda.synchronize()
    peak = torch.cuda.max_memory_allocated() - was
    assert peak <= max(cuda_ops().SCORED_BYTES, rows * Hq * 4) + (64 << 20), peak
    want, _, weights, mass, terms = attend(q, cache, md, 0.1)
    eps, u = weight_error(terms, 128), unit(q.dtype)
    assert ((out.double() - want).abs() <= u * want.abs() + (u * u + 2 * eps + 2.0 ** -13) * mass).all()
    total = before.double()
    total[:, :, :weights.shape[2]] += weights
    bound = 2.0 ** -24 * total
    bound[:, :, :weights.shape[2]] += (2 * eps + max(2.0 ** -20, Hq // Hkv * 2.0 ** -24)) * weights + 2.0 ** -126
    assert ((scores[:, :, :n].double() - total).abs() <= bound).all() and not scores[:, :, n:].any()


@pytest.mark.parametrize("vt", [True, False])
def test_decode_in_groups(vt, monkeypatch):
    """Requests of several launches, one workspace: as in one, to the bound of 64 bits; lengths of 0 among them."""
    lens = [300, 0, 17, 1000, 64, 5, 0, 130, 700, 33, 1]
    monkeypatch.setattr(cuda_ops(), "scored_parts", lambda *a: 0)
    for most in (1, 3, 4, 8):
        q, cache, md, scores = step(lens, [1] * len(lens), 8, 2, 128, 64, torch.bfloat16, "cuda", vt=vt, seed=8)
        monkeypatch.setattr(cuda_ops(), "SCORED_BYTES", most * 8 * 17 * 256)
        _check_decode(q, cache, md, scores, sinks=torch.randn(8, device="cuda"))


def test_weights_between_products():
    """Products on either side in the stream, whose tensor memory and that of the weights take turns: the same bits as by itself."""
    q, cache, md, scores = step([300, 64], [1, 1], 8, 2, 128, 64, torch.bfloat16, "cuda", vt=True)
    lse = torch.full((2, 8), 5.0, device="cuda")
    x, w = torch.randn(64, 1024, device="cuda").bfloat16(), torch.randn(1024, 1024, device="cuda").bfloat16()
    want = ops.key_weights(q, cache, md, 0.09, lse, scores.clone()), ops.linear(x, w), ops.paged_attention(q, cache, md, 0.09)
    for _ in range(200):
        got = [ops.linear(x, w), ops.key_weights(q, cache, md, 0.09, lse, scores.clone())]
        got += [ops.linear(x, w), ops.paged_attention(q, cache, md, 0.09), ops.key_weights(q, cache, md, 0.09, lse, scores.clone())]
        assert all(torch.equal(x, want[i]) for x, i in zip(got, (1, 0, 1, 2, 0)))


@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("D,BS,vt", [(128, 64, True), (64, 16, False)])
def test_one_row_of_a_wider_one(prompt, D, BS, vt):
    """A single query row out of rows of an odd width."""
    q, cache, md, scores = step([300], [1], 8, 2, D, BS, torch.bfloat16, "cuda", vt=vt)
    md.decode_only = not prompt
    lse, other = torch.full((1, 8), 5.0, device="cuda"), scores.clone()
    want = ops.scored_attention(q, cache, md, 0.1, other), ops.key_weights(q, cache, md, 0.1, lse, scores.clone())
    q = torch.nn.functional.pad(q.flatten(1), (0, 5)).expand(3, -1).contiguous()[:, :8 * D].unflatten(1, (8, D))[:1]
    assert q.is_contiguous() and q.stride(0) % 8
    assert torch.equal(ops.key_weights(q, cache, md, 0.1, lse, scores.clone()), want[1])
    assert torch.equal(ops.scored_attention(q, cache, md, 0.1, scores), want[0]) and torch.equal(scores, other)


FIRST = """
import torch
from tests.key_budget_oracle import step
from vllm_b200 import ops
lens = [300, 20, 1000]
q, cache, md, scores = step(lens, [1, 1, 1], 8, 2, 128, 64, torch.bfloat16, "cuda", vt=True, room=1030)
pq, _, pmd, _ = step([300], [40], 8, 2, 128, 64, torch.bfloat16, "cuda", room=1030)
pmd.block_table, pmd.seq_lens, pmd.kv_vt = md.block_table[:1], md.seq_lens[:1], True
lse, before, was = torch.full((40, 8), 6.0, device="cuda"), scores.clone(), cache.clone()
def call():
    out = ops.scored_attention(q, cache, md, 0.09, scores)
    ops.key_weights(pq, cache, pmd, 0.09, lse, scores, 30.0)
    return out, scores, cache, *ops.evict_keys(cache, md, scores, 200, 1, 9)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = call()
graph.replay()
got = [x.clone() for x in got]
scores.copy_(before), cache.copy_(was)
for x, y in zip(got, call()):
    assert torch.equal(x.view(torch.int16), y.view(torch.int16))
torch.cuda.synchronize()
print("same")
"""


def test_first_calls_in_a_capture():
    """A process whose first calls are captured: what is asked of the device once may be asked then."""
    got = subprocess.run([sys.executable, "-c", FIRST], capture_output=True, text=True, timeout=600, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert got.returncode == 0 and got.stdout.strip().endswith("same"), got.stderr[-2000:]


@pytest.mark.parametrize("vt", [True, False])
def test_pages_far_behind(vt):
    """Pages whose values lie more than 2^32 values into the cache."""
    q, cache, md, scores = step([300, 70, 700], [1, 1, 1], 8, 8, 128, 64, torch.bfloat16, "cuda", vt=vt, seed=9)
    far = 34000
    big = torch.empty(far + cache.shape[0], *cache.shape[1:], dtype=cache.dtype, device="cuda")
    big[far:] = cache
    shifted = dataclasses.replace(md, block_table=md.block_table + far)
    lse, keep = torch.full((3, 8), 5.0, device="cuda"), scores.clone()
    for call in (lambda c, m, s: ops.scored_attention(q, c, m, 0.1, s), lambda c, m, s: ops.key_weights(q, c, m, 0.1, lse, s),
                 lambda c, m, s: ops.scored_attention(q, c, dataclasses.replace(m, decode_only=False), 0.1, s), lambda c, m, s: ops.evict_keys(c, m, s, 100, 2, 9)):
        a, b = keep.clone(), keep.clone()
        want, got = call(cache, md, a), call(big, shifted, b)
        assert torch.equal(a, b)
        for x, y in zip(want if isinstance(want, tuple) else (want,), got if isinstance(got, tuple) else (got,)):
            assert torch.equal(x, y)
        assert torch.equal(cache.view(torch.int16), big[far:].view(torch.int16))
