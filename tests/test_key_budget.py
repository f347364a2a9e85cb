"""A key-value cache with a budget on the CPU: the plain forms against 64 bits, a run of the operators as a generation uses them, and what is refused."""
import dataclasses

import pytest
import torch

from tests.key_budget_oracle import attend, evict, step, unit, weight_error
from vllm_b200 import ops


@pytest.mark.parametrize("cap,sink,last", [(0.0, False, 0), (20.0, True, 3)])
@pytest.mark.parametrize("lens,queries", [([5, 33, 0, 16], [1, 1, 1, 1]), ([5, 33, 0, 40, 17], [5, 4, 0, 1, 17])])
def test_weights(lens, queries, cap, sink, last):
    q, cache, md, scores = step(lens, queries, 4, 2, 24, 16, torch.float32, "cpu")
    sinks = torch.randn(4) if sink else None
    if md.decode_only:
        last = 0
    want, norm, weights, mass, terms = attend(q, cache, md, 0.3, cap, sinks, last)
    before, eps = scores.clone(), weight_error(terms, 24)
    got = ops.scored_attention(q, cache, md, 0.3, scores, cap, sinks, last)
    assert ((got.double() - want).abs() <= 2.0 ** -24 * want.abs() + (2 * eps + 2.0 ** -18) * mass).all()
    n = weights.shape[2]
    assert ((scores - before)[:, :, :n].double() - weights).abs().max() <= 2.0 ** -24 * scores.max() * 2 + (2 * eps + 2.0 ** -18) * weights.max()
    assert torch.equal(scores[:, :, n:], before[:, :, n:])
    lse = norm.float()
    lse[0] = float("-inf")                              # a row without keys gives nothing
    again = ops.key_weights(q, cache, md, 0.3, lse, before.clone(), cap, last)
    more = attend(q, cache, md, 0.3, cap, sinks, last, torch.where(lse == float("-inf"), torch.inf, lse))[2]
    assert ((again - before)[:, :, :n].double() - more).abs().max() <= 2.0 ** -24 * again.max() * 2 + (2 * eps + 2.0 ** -18) * more.max()


CASES = [([5, 33, 0, 16], 10, 0, 0), ([5, 33, 0, 16], 33, 2, 3), ([40, 90], 1, 1, 0), ([40, 90, 64], 64, 4, 60), ([128], 127, 0, 1)]


@pytest.mark.parametrize("vt", [False, True])
@pytest.mark.parametrize("lens,keep,first,recent", CASES)
@pytest.mark.parametrize("kind", ["", "equal", "odd"])
def test_evict(lens, keep, first, recent, kind, vt):
    _, cache, md, scores = step(lens, [1] * len(lens), 4, 2, 128 if vt else 24, 64 if vt else 16, torch.float32, "cpu", vt=vt, seed=keep)
    if kind == "equal":
        scores = scores.round()
    if kind == "odd":
        scores[:, :, ::3], scores[:, :, 1::7], scores[:, :, 2::9] = float("nan"), float("inf"), -0.0
        scores[:, 1, 4::9] = float("-inf")
    positions = None
    for _ in range(2):
        want = evict(cache, md, scores, keep, first, recent, positions)
        got = ops.evict_keys(cache, md, scores, keep, first, recent, positions)
        assert torch.equal(cache.view(torch.int32), want[0].view(torch.int32))
        assert torch.equal(got[0], want[1]) and torch.equal(got[2], want[3])
        assert torch.equal(got[1].view(torch.int32), want[2].view(torch.int32))
        # again, some tokens later, from the order that the first eviction left
        grown = torch.minimum(got[0] + 4, md.seq_lens)
        scores, positions, md.seq_lens, keep = got[1] + torch.rand(scores.shape) * (torch.arange(scores.shape[2]) < grown[:, None, None]), got[2], grown, max(1, keep - 2)
        first, recent = min(first, keep), min(recent, keep - min(first, keep))


def test_generation():
    """A prompt, an eviction, tokens, an eviction, tokens: as attention over the rows that are kept, by their positions."""
    torch.manual_seed(3)
    H, G, D, BS, keep = 2, 2, 16, 16, 24
    q, cache, md, scores = step([50], [50], H * G, H, D, BS, torch.float64, "cpu", room=96, spare=4)
    scores, cache = scores.zero_(), cache.nan_to_num(0.0)
    md.block_table = torch.arange(cache.shape[0], dtype=torch.int32)[None]
    text = [[cache[r // BS, part, :, r % BS].clone() for r in range(50)] for part in (0, 1)]
    cache.zero_()
    for part in (0, 1):
        for r in range(50):
            cache[r // BS, part, :, r % BS] = text[part][r]
    ops.scored_attention(q, cache, md, 0.25, scores, last=8)
    total = [torch.zeros(50, dtype=torch.float64) for _ in range(H)]
    kept = [list(range(50)) for _ in range(H)]
    k = torch.stack(text[0])
    for h in range(H):
        a = torch.einsum("tgd,nd->gtn", q[-8:, h * G:h * G + G], k[:, h]) * 0.25
        total[h] += a.masked_fill(torch.arange(50) > torch.arange(42, 50)[:, None], float("-inf")).softmax(-1).sum((0, 1))
    positions, n = None, 50
    for _ in range(3):
        lens, scores, positions = ops.evict_keys(cache, md, scores, keep, 2, 6, positions)
        for h in range(H):
            old = kept[h]
            free = [p for p in old if 2 <= p < n - 6]
            free.sort(key=lambda p: (-float(total[h][p]), p))
            kept[h] = [p for p in old if p < 2 or p >= n - 6] + free[:keep - 8]
            assert sorted(kept[h]) == sorted(positions[0, h, :keep].tolist())
        md.seq_lens = lens
        for i in range(9):
            md.seq_lens = md.seq_lens + 1
            md.seq_lens_cpu, md.max_seq_len, md.max_query_len, md.decode_only = md.seq_lens, int(md.seq_lens), 1, True
            md.query_start_loc = md.query_start_loc_cpu = torch.tensor([0, 1])
            at, x = int(md.seq_lens) - 1, torch.randn(3, H, D, dtype=torch.float64)
            for part in (0, 1):
                cache[at // BS, part, :, at % BS] = x[part]
                text[part].append(x[part])
            q = torch.randn(1, H * G, D, dtype=torch.float64)
            out = ops.scored_attention(q, cache, md, 0.25, scores)
            for h in range(H):
                kept[h].append(n)
                total[h] = torch.cat([total[h], torch.zeros(1, dtype=torch.float64)])
                places = torch.tensor(kept[h])
                w = (q[0, h * G:h * G + G] @ torch.stack(text[0])[places, h].t() * 0.25).softmax(-1)
                total[h][places] += w.sum(0)
                assert (out[0, h * G:h * G + G] - w @ torch.stack(text[1])[places, h]).abs().max() < 1e-5      # (that path sums in 32 bits)
                assert (scores[0, h, :at + 1].double() - total[h][positions[0, h, :at + 1].long()]).abs().max() < 1e-4
            n += 1


def test_refusals():
    q, cache, md, scores = step([5, 33], [1, 1], 4, 2, 24, 16, torch.float32, "cpu")
    lse = torch.zeros(2, 4)
    for bad in (scores.double(), scores[:, :1], scores[:1], scores[..., :20], scores.transpose(1, 2), scores[0], scores.mT.contiguous().mT):
        for call in (lambda: ops.scored_attention(q, cache, md, 1.0, bad), lambda: ops.key_weights(q, cache, md, 1.0, lse, bad), lambda: ops.evict_keys(cache, md, bad, 4)):
            with pytest.raises(ValueError):
                call()
    for call in (lambda: ops.scored_attention(q[:, :3], cache, md, 1.0, scores), lambda: ops.scored_attention(q.double(), cache, md, 1.0, scores),
                 lambda: ops.scored_attention(q[..., :8], cache, md, 1.0, scores), lambda: ops.scored_attention(q[:1], cache, md, 1.0, scores),
                 lambda: ops.scored_attention(q, cache, md, 1.0, scores, sinks=torch.zeros(3)), lambda: ops.scored_attention(q, cache, md, 1.0, scores, last=-1),
                 lambda: ops.scored_attention(q, cache, md, 1.0, scores, out=q[:1]), lambda: ops.key_weights(q, cache, md, 1.0, lse[:1], scores),
                 lambda: ops.key_weights(q, cache, md, 1.0, lse.double(), scores), lambda: ops.key_weights(q, cache, md, 1.0, lse, scores, last=-1),
                 lambda: ops.evict_keys(cache, md, scores, 0), lambda: ops.evict_keys(cache, md, scores, 4, 3, 2), lambda: ops.evict_keys(cache, md, scores, 4, -1),
                 lambda: ops.evict_keys(cache, md, scores, 4, 0, -1), lambda: ops.evict_keys(cache, md, scores, 4, positions=torch.zeros(2, 2, 38)),
                 lambda: ops.evict_keys(cache, md, scores, 4, positions=torch.zeros(2, 2, 30, dtype=torch.int32))):
        with pytest.raises(ValueError):
            call()
    md.causal = False
    with pytest.raises(ValueError):
        ops.scored_attention(q, cache, md, 1.0, scores)


def test_numbers_above_32_bits():
    """A budget, a protected part or a window larger than any request."""
    q, cache, md, scores = step([5, 33], [5, 33], 4, 2, 24, 16, torch.float32, "cpu", vt=False)
    lse = torch.zeros(38, 4)
    want = ops.key_weights(q, cache, md, 1.0, lse, scores.clone())
    for last in (2 ** 31, 2 ** 32 + 1):
        assert torch.equal(ops.key_weights(q, cache, md, 1.0, lse, scores.clone(), last=last), want)
    for numbers in ((2 ** 31, 0, 0), (2 ** 32 + 4, 0, 0), (2 ** 34, 2 ** 32 + 1, 2 ** 32 + 1)):
        was = cache.clone()
        lens, new, _ = ops.evict_keys(cache, md, scores, *numbers)
        assert lens.tolist() == [5, 33] and lens.dtype is torch.int32 and torch.equal(cache.view(torch.int32), was.view(torch.int32))
        assert torch.equal(new[1, :, :33], scores[1, :, :33])


def test_weights_infinite():
    """Rows whose log-sum-exp is infinite or NaN give nothing, whatever their scores are."""
    q, cache, md, scores = step([40], [9], 4, 2, 24, 16, torch.float32, "cpu")
    lse = attend(q, cache, md, 0.3)[1].float()
    want = ops.key_weights(q[5:], cache, dataclasses.replace(md, query_start_loc=torch.tensor([0, 4]), query_start_loc_cpu=torch.tensor([0, 4])), 0.3, lse[5:], scores.clone())
    lse[0], lse[1], lse[2:5] = float("nan"), float("-inf"), float("inf")
    q[3] = float("inf")
    assert torch.equal(ops.key_weights(q, cache, md, 0.3, lse, scores.clone()), want)
