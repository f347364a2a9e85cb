"""A key-value cache with a budget on the device: values, shapes and calls at the edge of what the operators take."""
import dataclasses

import pytest
import torch

from tests.key_budget_oracle import step
from tests.test_key_budget_gpu import _check_weights
from vllm_b200 import ops

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
