"""A key-value cache with a budget on the device: scored attention, key weights and eviction against 64 bits."""
import dataclasses

import pytest
import torch

from tests.key_budget_oracle import attend, evict, step, unit, weight_error
from vllm_b200 import ops
from vllm_b200.ops import cuda_ops

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
    # each weight as exact as its exponential and the log-sum-exp; an addition for every head of a kv head; the sum is rounded once
    bound = 2.0 ** -24 * total + 0.0
    bound[:md.num_reqs, :, :n] += (2 * eps + max(2.0 ** -20, q.shape[1] // cache.shape[2] * 2.0 ** -24)) * weights + 2.0 ** -126
    assert ((scores.double() - total).abs() <= bound).all(), ((scores.double() - total).abs() / bound.clamp(min=1e-300)).max()
    seen = torch.arange(scores.shape[2], device="cuda") < md.seq_lens[:md.num_reqs, None, None]
    assert torch.equal(scores[:md.num_reqs][~seen.expand_as(scores[:md.num_reqs])], before[:md.num_reqs][~seen.expand_as(scores[:md.num_reqs])])
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,D,BS,vt", [(8, 2, 128, 64, True), (16, 1, 128, 64, True), (3, 3, 128, 64, True), (10, 2, 64, 16, False), (24, 2, 64, 32, False),
                                            (6, 6, 80, 16, False), (8, 2, 96, 48, False), (20, 1, 128, 32, False), (40, 1, 128, 64, True), (4, 2, 256, 64, False),
                                            (16, 1, 256, 16, False), (2, 1, 8, 16, False), (5, 1, 72, 128, False)])
@pytest.mark.parametrize("cap,sink", [(0.0, False), (30.0, True)])
@pytest.mark.parametrize("runs", [False, True])
def test_decode(dtype, Hq, Hkv, D, BS, vt, cap, sink, runs, monkeypatch):
    """In clusters where the sizes allow it, and in runs of equal length."""
    if runs:
        monkeypatch.setattr(cuda_ops(), "scored_parts", lambda *a: 0)
    q, cache, md, scores = step(LENS, [1] * len(LENS), Hq, Hkv, D, BS, dtype, "cuda", vt=vt, seed=Hq + D, spread=2.0)
    sinks = torch.randn(Hq, device="cuda") if sink else None
    _check_decode(q, cache, md, scores, cap, sinks)


@pytest.mark.parametrize("lens", [[1], [0], [0, 40, 0, 0, 7, 0], [5000], [2048], [2047, 130], [64, 0, 65], [64] * 200, [1] * 700, [17000, 3, 9001], [2000] * 40, [700] * 3 + [0] * 1100 + [33] * 2])
@pytest.mark.parametrize("vt", [True, False])
@pytest.mark.parametrize("room", [0, 2048])
def test_decode_lengths(lens, vt, room):
    Hq, Hkv = (32, 8) if len(lens) < 300 else (2, 1)
    q, cache, md, scores = step(lens, [1] * len(lens), Hq, Hkv, 128, 64, torch.bfloat16, "cuda", vt=vt, seed=len(lens), room=max(room, max(lens) + 5))
    if room:                                  # a table for as many rows
        md.block_table = torch.nn.functional.pad(md.block_table, (0, max(0, 32 - md.block_table.shape[1])))
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


@pytest.mark.parametrize("n,keep", [(4096, 1000), (4097, 4000), (9000, 100), (33000, 8000), (33000, 32990), (400000, 3000), (450000, 2000)])
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


@pytest.mark.parametrize("told", [1, 4000])
def test_weights_with_another_maximum(told):
    """The longest query of the metadata only chooses how the work is dealt out."""
    q, cache, md, scores = step([1500, 700], [1500, 300], 8, 2, 128, 64, torch.bfloat16, "cuda", vt=True)
    md.max_query_len = told
    _check_weights(q, cache, md, scores)


def test_weights_of_rows_without():
    """Rows whose log-sum-exp says that they have no key, or is NaN, give nothing."""
    q, cache, md, scores = step([300, 200], [100, 200], 8, 2, 128, 64, torch.bfloat16, "cuda", seed=1)
    lse = attend(q, cache, md, 128 ** -0.5)[1].float()
    lse[::3], lse[1::5] = float("-inf"), float("nan")
    _check_weights(q, cache, md, scores, lse=lse)


def test_evict_nothing():
    _, cache, md, scores = step([0, 0], [1, 1], 2, 2, 64, 16, torch.bfloat16, "cuda")
    _check_evict(cache, md, scores, 4, 1, 1)
    got = ops.evict_keys(cache, md, scores[..., :0], 4)
    assert got[0].tolist() == [0, 0] and got[1].shape == got[2].shape == (2, 2, 0)


@pytest.mark.parametrize("kind", ["queries", "scores", "out", "table"])
def test_strides(kind):
    """Queries out of a merged projection, scores of more requests and rows than there are, an output with other columns, a wider table."""
    lens = [300, 17, 64]
    q, cache, md, scores = step(lens, [1, 1, 1], 8, 2, 128, 64, torch.bfloat16, "cuda", vt=True, seed=3)
    out = None
    if kind == "queries":
        q = torch.cat([torch.randn(3, 3, 128, device="cuda").bfloat16(), q, torch.randn(3, 2, 128, device="cuda").bfloat16()], 1)[:, 3:11]
    if kind == "scores":
        big = torch.rand(7, 4, 999, device="cuda")
        big[:, :2, :scores.shape[2]][:3] = scores
        rest = big.clone()
        scores = big[:, :2, :scores.shape[2]]
    if kind == "out":
        out = torch.zeros(3, 20, 128, device="cuda", dtype=torch.bfloat16)[:, 5:13]
    if kind == "table":
        md.block_table = torch.cat([md.block_table, torch.full((3, 9), -7, dtype=torch.int32, device="cuda")], 1)[:, :md.block_table.shape[1] + 3]
    got = _check_decode(q, cache, md, scores, out=out)
    if kind == "out":
        assert got is out
    if kind == "scores":
        assert torch.equal(big[3:], rest[3:]) and torch.equal(big[:, 2:], rest[:, 2:]) and torch.equal(big[:, :, scores.shape[2]:], rest[:, :, scores.shape[2]:])
    _check_weights(q, cache, md, scores[:3])
    if kind == "scores":
        moved = torch.arange(999, device="cuda", dtype=torch.int32).expand(7, 4, 999).contiguous()[:3, :2, :scores.shape[2]]
        _check_evict(cache, md, scores[:3], 50, 2, 3, moved)


def test_padding_rows():
    """A batch that is padded to a bucket: rows behind the requests are zeros, their scores as they were."""
    q, cache, md, scores = step([70, 33], [1, 1], 8, 2, 128, 64, torch.bfloat16, "cuda", vt=True)
    q = torch.cat([q, torch.full_like(q, float("nan"))])
    scores = torch.cat([scores, torch.rand_like(scores)])
    before = scores[2:].clone()
    got = _check_decode(q, cache, md, scores)
    assert got.shape == q.shape and not got[2:].any() and torch.equal(scores[2:], before)


def test_bad_tables():
    """Numbers of pages that the cache does not have: whatever comes out, nothing outside the cache is read or written."""
    q, cache, md, scores = step([300, 40], [1, 1], 8, 2, 128, 64, torch.bfloat16, "cuda", vt=True)
    whole = torch.full((cache.shape[0] + 8, *cache.shape[1:]), 3.0, dtype=cache.dtype, device="cuda")
    whole[4:-4] = cache
    md.block_table[0, 1], md.block_table[0, 2], md.block_table[1, 0] = 1 << 30, -5, cache.shape[0]
    cache = whole[4:-4]
    ops.scored_attention(q, cache, md, 0.1, scores)
    ops.key_weights(q, cache, md, 0.1, torch.zeros(2, 8, device="cuda"), scores)
    ops.evict_keys(cache, md, torch.rand_like(scores), 100)
    torch.cuda.synchronize()
    assert (whole[:4] == 3).all() and (whole[-4:] == 3).all()


@pytest.mark.parametrize("vt", [True, False])
def test_generation(vt):
    """A prompt, an eviction, tokens, an eviction, tokens: against the same with 64 bits, by the rows' positions."""
    H, G, D, BS, keep = 2, 4, 128, 64, 150
    lens = [400, 90, 260]
    q, cache, md, scores = step(lens, lens, H * G, H, D, BS, torch.bfloat16, "cuda", vt=vt, room=700, spare=40)
    scores.zero_()
    md.block_table = torch.cat([md.block_table, torch.zeros(3, 6, dtype=torch.int32, device="cuda")], 1)
    used = set(md.block_table[torch.arange(md.block_table.shape[1], device="cuda") < torch.tensor([[-(-n // BS)] for n in lens], device="cuda")].tolist())
    free = [b for b in range(cache.shape[0]) if b not in used]
    for b, n in enumerate(lens):
        for i in range(-(-n // BS), md.block_table.shape[1]):
            md.block_table[b, i] = free.pop()
    cache.nan_to_num_(0.0)
    want_scores = scores.double()
    want_scores[:, :, :400] += attend(q, cache, md, D ** -0.5, last=32)[2]
    ops.scored_attention(q, cache, md, D ** -0.5, scores, last=32)
    assert (scores.double() - want_scores).abs().max() < 2e-3               # (the prompt's log-sum-exps are those of weights in 16 bits)
    values = cache[:, 1].view(-1, H, D, BS).transpose(2, 3) if vt else cache[:, 1]
    positions, total = None, torch.tensor(lens, device="cuda")
    for _ in range(3):
        md.max_seq_len = int(md.seq_lens.max())
        new, scores, positions = _check_evict(cache, md, scores, keep, 2, 20, positions)
        assert torch.equal(positions[:, 0].gather(1, new[:, None].long())[:, 0], total.int())      # of the next token
        md.seq_lens = new
        for _ in range(30):
            md.seq_lens = md.seq_lens + 1
            total = total + 1
            md.query_start_loc, md.max_query_len, md.decode_only, md.max_seq_len = torch.arange(4, dtype=torch.int32, device="cuda"), 1, True, int(md.seq_lens.max())
            for b, n in enumerate(md.seq_lens.tolist()):
                page = int(md.block_table[b, (n - 1) // BS])
                cache[page, 0, :, (n - 1) % BS] = torch.randn(H, D, device="cuda")
                values[page, :, (n - 1) % BS] = torch.randn(H, D, device="cuda").bfloat16()
            _check_decode(torch.randn(3, H * G, D, device="cuda").bfloat16(), cache, md, scores)
    assert int(md.seq_lens.max()) == keep + 30


def test_graphs():
    """Captured steps, replayed in turn with other inputs than they were captured with, beside the same calls on another stream."""
    calls, graphs = [], []
    for k, lens in enumerate([[300, 20, 1000], [64, 900, 5]]):
        q, cache, md, scores = step(lens, [1, 1, 1], 8, 2, 128, 64, torch.bfloat16, "cuda", vt=True, seed=k, room=1030)
        md.max_seq_len = 1030
        pq, _, pmd, _ = step([n for n in lens], [min(n, 40) for n in lens], 8, 2, 128, 64, torch.bfloat16, "cuda", seed=9)
        pmd = dataclasses.replace(pmd, block_table=md.block_table, seq_lens=md.seq_lens, kv_vt=True)
        lse = torch.full((pq.shape[0], 8), 6.0, device="cuda")

        def call(q=q, cache=cache, md=md, scores=scores, pq=pq, pmd=pmd, lse=lse):
            out = ops.scored_attention(q, cache, md, 0.09, scores)
            ops.key_weights(pq, cache, pmd, 0.09, lse, scores)
            return out, scores, cache, *ops.evict_keys(cache, md, scores, 200, 1, 9)
        calls.append((call, q, scores, cache))
    for call, _, scores, cache in calls:
        keep = scores.clone(), cache.clone()
        call()                                           # (what is compiled or looked up at a first call)
        scores.copy_(keep[0]), cache.copy_(keep[1])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for turn in range(3):
        for (call, q, scores, cache), (g, out) in zip(calls, graphs):
            q.copy_(torch.randn(q.shape, device="cuda"))
            scores.copy_(torch.rand_like(scores) * (scores > 0))
            keep = scores.clone(), cache.clone()
            want = [x.clone() for x in call()]
            scores.copy_(keep[0]), cache.copy_(keep[1])
            g.replay()
            torch.cuda.synchronize()
            for x, y in zip(out, want):
                assert torch.equal(x.view(torch.int16), y.view(torch.int16))
            scores.copy_(keep[0]), cache.copy_(keep[1])
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    wants, gots = [], []
    for call, _, scores, cache in calls:
        keep = scores.clone(), cache.clone()
        wants.append([x.clone() for x in call()])
        scores.copy_(keep[0]), cache.copy_(keep[1])
    torch.cuda.synchronize()
    for (call, *_), stream in zip(calls, streams):
        with torch.cuda.stream(stream):
            gots.append(call())
    torch.cuda.synchronize()
    for got, want in zip(gots, wants):
        assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip(got, want))


@pytest.mark.parametrize("vt", [True, False])
def test_batch_invariant(vt, monkeypatch):
    """In that mode a request's output and scores have the same bits alone and in a batch."""
    monkeypatch.setenv("VLLM_BATCH_INVARIANT", "1")
    lens = [700, 33, 1500]
    for queries in ([1, 1, 1], [200, 33, 1]):
        q, cache, md, scores = step(lens, queries, 8, 2, 128, 64, torch.bfloat16, "cuda", vt=vt, seed=4)
        each = scores.clone()
        out = ops.scored_attention(q, cache, md, 0.1, scores)
        start = md.query_start_loc.tolist()
        for b, n in enumerate(lens):
            one = dataclasses.replace(md, num_reqs=1, num_actual_tokens=queries[b], max_query_len=queries[b], max_seq_len=n, decode_only=queries[b] == 1,
                                      query_start_loc=torch.tensor([0, queries[b]], dtype=torch.int32, device="cuda"), seq_lens=md.seq_lens[b:b + 1].clone(),
                                      block_table=md.block_table[b:b + 1])
            alone = ops.scored_attention(q[start[b]:start[b + 1]].clone(), cache, one, 0.1, each[b:b + 1])
            assert torch.equal(alone, out[start[b]:start[b + 1]]) and torch.equal(each[b], scores[b])


def test_same_bits():
    q, cache, md, scores = step([5000, 300, 17], [1, 1, 1], 32, 8, 128, 64, torch.bfloat16, "cuda", vt=True)
    pq, pcache, pmd, pscores = step([3000, 300], [3000, 300], 32, 8, 128, 64, torch.bfloat16, "cuda")
    lse = torch.full((3300, 32), 7.0, device="cuda")
    want = None
    for _ in range(5):
        s, t = scores.clone(), pscores.clone()
        got = ops.scored_attention(q, cache, md, 0.1, s), s, ops.key_weights(pq, pcache, pmd, 0.1, lse, t)
        assert want is None or all(torch.equal(a, b) for a, b in zip(got, want))
        want = got


def test_numbers_above_32_bits():
    q, cache, md, scores = step([5, 300], [5, 300], 8, 2, 128, 64, torch.bfloat16, "cuda")
    lse = torch.full((305, 8), 3.0, device="cuda")
    want = ops.key_weights(q, cache, md, 0.1, lse, scores.clone())
    for last in (2 ** 31, 2 ** 32 + 1):
        assert torch.equal(ops.key_weights(q, cache, md, 0.1, lse, scores.clone(), last=last), want)
    for numbers in ((2 ** 31, 0, 0), (2 ** 32 + 4, 0, 0), (2 ** 34, 2 ** 32 + 1, 2 ** 32 + 1)):
        was = cache.clone()
        lens, new, _ = ops.evict_keys(cache, md, scores, *numbers)
        assert lens.tolist() == [5, 300] and torch.equal(cache.view(torch.int16), was.view(torch.int16)) and torch.equal(new[1, :, :300], scores[1, :, :300])


@pytest.mark.parametrize("Hq,D,BS", [(256, 64, 16), (255, 128, 64)])
def test_decode_many_heads(Hq, D, BS):
    q, cache, md, scores = step([1, 200, 70], [1] * 3, Hq, 1, D, BS, torch.bfloat16, "cuda", spread=2.0)
    _check_decode(q, cache, md, scores)


def test_step_refusals():
    """What a step says of its requests: too few of them, or on the host."""
    q, cache, md, scores = step([33, 5], [1, 1], 8, 2, 128, 64, torch.bfloat16, "cuda", vt=True)
    lse = torch.zeros(2, 8, device="cuda")
    replace = dataclasses.replace
    for md_ in (replace(md, block_table=md.block_table.cpu()), replace(md, seq_lens=md.seq_lens.cpu()), replace(md, block_table=md.block_table[:1]),
                replace(md, seq_lens=md.seq_lens[:1]), replace(md, block_table=md.block_table[0])):
        for call in (lambda: ops.scored_attention(q, cache, md_, 0.1, scores), lambda: ops.key_weights(q, cache, md_, 0.1, lse, scores),
                     lambda: ops.evict_keys(cache, md_, scores, 4)):
            with pytest.raises(ValueError):
                call()
    for qsl in (md.query_start_loc[:2], md.query_start_loc.cpu()):
        with pytest.raises(ValueError):
            ops.key_weights(q, cache, replace(md, decode_only=False, query_start_loc=qsl), 0.1, lse, scores)
    many = step([33, 5], [1, 1], 257, 1, 64, 16, torch.bfloat16, "cuda")
    with pytest.raises(ValueError):
        ops.scored_attention(many[0], many[1], many[2], 0.1, many[3])


def test_refusals(monkeypatch):
    q, cache, md, scores = step([33, 5], [1, 1], 8, 2, 128, 64, torch.bfloat16, "cuda", vt=True)
    lse = torch.zeros(2, 8, device="cuda")
    replace = dataclasses.replace
    bad_table, bad_lens = replace(md, block_table=md.block_table.long()), replace(md, seq_lens=md.seq_lens.long())
    cases = [(q.float(), cache.float(), md), (q, cache.to(torch.float8_e4m3fn), md), (q, cache, bad_table), (q, cache, bad_lens), (q[..., :64], cache[..., :64], md),
             (q, cache.transpose(1, 2).contiguous().transpose(1, 2), md)]
    small = step([33, 5], [1, 1], 8, 2, 64, 16, torch.bfloat16, "cuda")
    cases += [(small[0], small[1], replace(small[2], kv_vt=True)), (small[0][..., :60], small[1][..., :60].contiguous(), small[2])]
    odd = torch.zeros(cache.numel() + 4, dtype=cache.dtype, device="cuda")[4:].view(cache.shape)
    cases += [(q, odd, md), (q, cache[:, :, :, :40].contiguous(), replace(md, kv_vt=False))]
    for q_, cache_, md_ in cases:
        for call in (lambda: ops.scored_attention(q_, cache_, md_, 0.1, scores), lambda: ops.key_weights(q_, cache_, md_, 0.1, lse, scores),
                     lambda: ops.evict_keys(cache_, md_, scores, 4)):
            with pytest.raises(ValueError):
                call()
    with pytest.raises(ValueError):
        ops.key_weights(q, cache, md, 0.0, lse, scores)
    with pytest.raises(ValueError):
        ops.scored_attention(q, cache, md, 0.1, scores, out=q.transpose(0, 1).contiguous().transpose(0, 1))
    with pytest.raises(ValueError):
        ops.key_weights(q, cache, replace(md, decode_only=False, query_start_loc=md.query_start_loc.long()), 0.1, lse, scores)
    many = step([33, 5], [1, 1], 129, 1, 64, 16, torch.bfloat16, "cuda")
    with pytest.raises(ValueError):
        ops.key_weights(many[0], many[1], many[2], 0.1, torch.zeros(2, 129, device="cuda"), many[3])
    from vllm_b200.ops import cuda as cu
    monkeypatch.setattr(cu, "_device", lambda: 1)
    with pytest.raises(ValueError):
        ops.scored_attention(q, cache, md, 0.1, scores)
