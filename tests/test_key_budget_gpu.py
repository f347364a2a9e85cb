"""A key-value cache with a budget on the device: scored attention, key weights and eviction against 64 bits."""
import pytest
import torch

from tests.key_budget_oracle import attend, step, unit, weight_error
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
