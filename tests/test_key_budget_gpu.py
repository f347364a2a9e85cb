"""A key-value cache with a budget on the device: scored attention, key weights and eviction against 64 bits."""
import dataclasses

import pytest
import torch

from tests.key_budget_oracle import attend, evict, step, unit, weight_error
from vllm_b200 import ops

pytestmark = pytest.mark.gpu
LENS = [1, 15, 16, 17, 63, 64, 65, 300, 1030]


def _check_decode(q, cache, md, scores, cap=0.0, sinks=None, scale=None, out=None):
    D = q.shape[2]
    scale = D ** -0.5 if scale is None else scale
    want, _, weights, mass, terms = attend(q[:md.num_reqs], cache, md, scale, cap, sinks)
    before = scores.clone()
    got = ops.scored_attention(q, cache, md, scale, scores, logits_soft_cap=cap, sinks=sinks, out=out)
    eps, u = weight_error(terms, D), unit(q.dtype)
    # weights in two 16-bit parts, 32-bit sums of up to 2^11 keys a warp, the result rounded once (fp16: to multiples of 2^-24)
    bound = u * want.abs() + (u * u + 2 * eps + 2.0 ** -13) * mass + (2.0 ** -25 if q.dtype is torch.float16 else 0.0)
    assert ((got[:md.num_reqs].double() - want).abs() <= bound).all(), ((got[:md.num_reqs].double() - want).abs() / bound).max()
    n = weights.shape[2]
    total = before.double()
    total[:md.num_reqs, :, :n] += weights
    # each weight as exact as its exponential and the log-sum-exp; the sum is rounded once
    bound = 2.0 ** -24 * total + 0.0
    bound[:md.num_reqs, :, :n] += (2 * eps + 2.0 ** -20) * weights + 2.0 ** -126
    assert ((scores.double() - total).abs() <= bound).all(), ((scores.double() - total).abs() / bound.clamp(min=1e-300)).max()
    seen = torch.arange(scores.shape[2], device="cuda") < md.seq_lens[:md.num_reqs, None, None]
    assert torch.equal(scores[:md.num_reqs][~seen.expand_as(scores[:md.num_reqs])], before[:md.num_reqs][~seen.expand_as(scores[:md.num_reqs])])
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,D,BS,vt", [(8, 2, 128, 64, True), (16, 1, 128, 64, True), (3, 3, 128, 64, True), (10, 2, 64, 16, False), (24, 2, 64, 32, False),
                                            (6, 6, 80, 16, False), (8, 2, 96, 48, False), (20, 1, 128, 32, False), (40, 1, 128, 64, True), (4, 2, 256, 64, False),
                                            (16, 1, 256, 16, False), (2, 1, 8, 16, False), (5, 1, 72, 128, False)])
@pytest.mark.parametrize("cap,sink", [(0.0, False), (30.0, True)])
def test_decode(dtype, Hq, Hkv, D, BS, vt, cap, sink):
    q, cache, md, scores = step(LENS, [1] * len(LENS), Hq, Hkv, D, BS, dtype, "cuda", vt=vt, seed=Hq + D, spread=2.0)
    sinks = torch.randn(Hq, device="cuda") if sink else None
    _check_decode(q, cache, md, scores, cap, sinks)


@pytest.mark.parametrize("lens", [[1], [0], [0, 40, 0, 0, 7, 0], [5000], [64] * 200, [1] * 700, [17000, 3, 9001], [2000] * 40, [700] * 3 + [0] * 1100 + [33] * 2])
@pytest.mark.parametrize("vt", [True, False])
def test_decode_lengths(lens, vt):
    Hq, Hkv = (32, 8) if len(lens) < 300 else (2, 1)
    q, cache, md, scores = step(lens, [1] * len(lens), Hq, Hkv, 128, 64, torch.bfloat16, "cuda", vt=vt, seed=len(lens))
    _check_decode(q, cache, md, scores)


def _check_evict(cache, md, scores, keep, first=0, recent=0, positions=None):
    want = evict(cache.cpu(), _on_cpu(md), scores.cpu(), keep, first, recent, None if positions is None else positions.cpu())
    got = ops.evict_keys(cache, md, scores, keep, first, recent, positions)
    assert torch.equal(got[0].cpu(), want[1]) and torch.equal(got[2].cpu(), want[3])
    assert torch.equal(got[1].cpu().view(torch.int32), want[2].view(torch.int32))
    assert torch.equal(cache.cpu().view(torch.int16), want[0].view(torch.int16))
    return got


def _on_cpu(md):
    return dataclasses.replace(md, block_table=md.block_table.cpu(), seq_lens=md.seq_lens.cpu())


@pytest.mark.parametrize("D,BS,vt,dtype", [(128, 64, True, torch.bfloat16), (128, 64, False, torch.float16), (64, 16, False, torch.bfloat16), (80, 48, False, torch.bfloat16),
                                           (256, 32, False, torch.float16), (8, 16, False, torch.bfloat16)])
@pytest.mark.parametrize("lens,keep,first,recent", [([5, 33, 0, 16], 10, 0, 0), ([5, 33, 0, 16], 33, 2, 3), ([40, 90], 1, 1, 0), ([40, 900, 64], 64, 4, 60), ([128], 127, 0, 1),
                                                    ([1500, 31, 777], 512, 4, 100), ([4500], 4000, 0, 0)])
@pytest.mark.parametrize("kind", ["", "equal", "odd"])
def test_evict(D, BS, vt, dtype, lens, keep, first, recent, kind):
    Hkv = 3 if vt else 2
    _, cache, md, scores = step(lens, [1] * len(lens), Hkv, Hkv, D, BS, dtype, "cuda", vt=vt, seed=keep)
    if kind == "equal":
        scores = scores.round()
    if kind == "odd":
        scores[:, :, ::3], scores[:, :, 1::7], scores[:, :, 2::9] = float("nan"), float("inf"), -0.0
        scores[:, 1, 4::9], scores[:, 0] = float("-inf"), -scores[:, 0]
    new, positions = None, None
    for _ in range(2):
        new, scores, positions = _check_evict(cache, md, scores, keep, first, recent, positions)
        grown = torch.minimum(new + 4, md.seq_lens)
        scores += torch.rand_like(scores) * (torch.arange(scores.shape[2], device="cuda") < grown[:, None, None])
        md.seq_lens, keep = grown, max(1, keep - 2)
        first, recent = min(first, keep), min(recent, keep - min(first, keep))


@pytest.mark.parametrize("n,keep", [(4096, 1000), (4097, 4000), (9000, 100), (33000, 8000), (33000, 32990), (450000, 2000)])
def test_evict_long(n, keep):
    """A request of a cluster, and one that its shared memory does not hold."""
    _, cache, md, scores = step([n, n // 3], [1, 1], 2, 2, 8, 64, torch.bfloat16, "cuda", seed=n)
    _, scores, positions = _check_evict(cache, md, scores, keep, 3, 50)
    md.seq_lens = torch.clamp(md.seq_lens, max=keep)
    _check_evict(cache, md, scores, keep // 2, 1, 20, positions)


def _check_weights(q, cache, md, scores, cap=0.0, last=0, scale=None, lse=None):
    D = q.shape[2]
    scale = D ** -0.5 if scale is None else scale
    if lse is None:
        lse = attend(q, cache, md, scale, cap)[1].float()
    _, _, weights, _, terms = attend(q, cache, md, scale, cap, None, last, torch.where(lse > float("-inf"), lse, torch.inf))
    before = scores.clone()
    assert ops.key_weights(q, cache, md, scale, lse, scores, cap, last) is scores
    n = weights.shape[2]
    total = before.double()
    total[:, :, :n] += weights
    # each weight as exact as its exponential; 128 columns are added in chains of 34, their sums without loss; the last addition is rounded
    bound = 2.0 ** -24 * total
    bound[:, :, :n] += (weight_error(terms, D) + 38 * 2.0 ** -24) * weights + 2.0 ** -126
    assert ((scores.double() - total).abs() <= bound).all(), ((scores.double() - total).abs() / bound.clamp(min=1e-300)).max()
    seen = torch.arange(scores.shape[2], device="cuda") < md.seq_lens[:, None, None]
    assert torch.equal(scores[~seen.expand_as(scores)], before[~seen.expand_as(scores)])


SHAPES = [(8, 2, 128, 64, True), (16, 1, 128, 64, True), (3, 3, 128, 64, True), (10, 2, 64, 16, False), (24, 2, 64, 32, False), (6, 6, 80, 16, False), (8, 2, 96, 48, False),
          (40, 1, 128, 128, False), (4, 2, 256, 64, False), (16, 1, 192, 256, False), (2, 1, 8, 16, False), (128, 1, 72, 16, False)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,D,BS,vt", SHAPES)
@pytest.mark.parametrize("cap,last", [(0.0, 0), (30.0, 5), (0.0, 64)])
def test_weights(dtype, Hq, Hkv, D, BS, vt, cap, last):
    lens, queries = [300, 1, 700, 0, 64, 130, 511, 513], [300, 1, 45, 0, 1, 129, 256, 3]
    q, cache, md, scores = step(lens, queries, Hq, Hkv, D, BS, dtype, "cuda", vt=vt, seed=Hq + D, spread=2.0)
    _check_weights(q, cache, md, scores, cap, last)


@pytest.mark.parametrize("lens,queries,last", [([1], [1], 0), ([2500], [2500], 0), ([2500], [2500], 64), ([9000, 300], [20, 300], 0), ([40] * 130, [40] * 130, 7),
                                               ([200, 300, 1000], [1, 1, 1], 0), ([257, 256, 255], [257, 256, 255], 1)])
def test_weights_lengths(lens, queries, last):
    q, cache, md, scores = step(lens, queries, 8, 2, 128, 64, torch.bfloat16, "cuda", vt=True, seed=len(lens))
    _check_weights(q, cache, md, scores, last=last)


def test_weights_of_rows_without():
    """Rows whose log-sum-exp says that they have no key, or is NaN, give nothing."""
    q, cache, md, scores = step([300, 200], [100, 200], 8, 2, 128, 64, torch.bfloat16, "cuda", seed=1)
    lse = attend(q, cache, md, 128 ** -0.5)[1].float()
    lse[::3], lse[1::5] = float("-inf"), float("nan")
    _check_weights(q, cache, md, scores, lse=lse)
