"""Scored attention of prompts and of batch-invariant mode: what a call says is looked at before anything is launched.  Runs on the host: the launches
are stand-ins that note that they were reached."""
import dataclasses

import pytest
import torch

from tests.key_budget_oracle import step
from vllm_b200 import ops
from vllm_b200.ops import cuda as cu


@pytest.fixture
def calls(monkeypatch):
    """Names of what was launched, in order, with the queries and the output that each was given."""
    seen = []

    def attention(q, kv_cache, md, scale, window=None, cap=0.0, causal=True, out=None, return_lse=False, sinks=None, **_):
        seen.append(("attention", q, out))
        used = md.num_reqs if md.decode_only else int(md.query_start_loc[-1])
        out = torch.full_like(q, float("nan"), memory_format=torch.contiguous_format) if out is None else out
        out[:used] = 2 * q[:used]                                               # (something that is exact)
        return out, torch.zeros(q.shape[:2])

    def weights(*a):
        seen.append(("weights",))
        return 0

    def decode(*a):
        seen.append(("decode",))
        return 0
    monkeypatch.setattr(ops, "_use_cuda", lambda x: True)
    for name, f in (("paged_attention", attention), ("_key_weights", weights), ("_scored_decode", decode), ("_device", lambda: -1), ("_st", lambda: 0),
                    ("num_sms", lambda: 148), ("_error_flag", lambda d: None)):
        monkeypatch.setattr(cu, name, f)
    return seen


def _steps(invariant, monkeypatch, Hq=8, Hkv=2, D=24, BS=16, vt=False):
    """A prompt, or a decode step in batch-invariant mode."""
    if invariant:
        monkeypatch.setenv("VLLM_BATCH_INVARIANT", "1")
    queries = [1, 1] if invariant else [20, 5]
    q, cache, md, scores = step([33, 5], queries, Hq, Hkv, D, BS, torch.bfloat16, "cpu", vt=vt)
    return q, cache.nan_to_num(0.0), md, scores


@pytest.mark.parametrize("invariant", [False, True])
def test_refusals(calls, monkeypatch, invariant):
    q, cache, md, scores = _steps(invariant, monkeypatch)
    replace = dataclasses.replace
    odd = torch.zeros(cache.numel() + 4, dtype=cache.dtype)[4:].view(cache.shape)
    assert odd.data_ptr() % 16 or cache.data_ptr() % 16
    bad = [(q, odd if odd.data_ptr() % 16 else cache, md, {})]
    for change in (dict(block_table=md.block_table.long()), dict(block_table=md.block_table[:1]), dict(block_table=md.block_table[0]), dict(block_table=md.block_table.t().contiguous().t()),
                   dict(seq_lens=md.seq_lens.long()), dict(seq_lens=md.seq_lens[:1]), dict(query_start_loc=md.query_start_loc.long()),
                   dict(query_start_loc=md.query_start_loc[:2]),
                   dict(block_table=md.block_table[:, :2])):                      # (two pages of 16 for 33 rows)
        bad.append((q, cache, replace(md, **change), {}))
    if not invariant:
        bad.append((q, cache, replace(md, query_start_loc=None), {}))
    bad.append((q, cache, md, {"out": q.transpose(0, 1).contiguous().transpose(0, 1)}))
    bad.append((q, cache, md, {"scale": 0.0}))
    for q_, cache_, md_, more in bad:
        more = {"scale": 0.1, **more}
        with pytest.raises(ValueError):
            ops.scored_attention(q_, cache_, md_, more.pop("scale"), scores, **more)
        assert not calls, (calls, md_, more)
    q, cache, md, scores = _steps(invariant, monkeypatch, Hq=129, Hkv=1)
    with pytest.raises(ValueError):
        ops.scored_attention(q, cache, md, 0.1, scores)
    for heads in (5, 40):                                                       # transposed values: 128 is no multiple of the heads of a kv head
        q, cache, md, scores = _steps(invariant, monkeypatch, Hq=heads, Hkv=1, D=128, BS=64, vt=True)
        with pytest.raises(ValueError):
            ops.scored_attention(q, cache, md, 0.1, scores)
    assert not calls


@pytest.mark.parametrize("invariant", [False, True])
@pytest.mark.parametrize("where", ["", "given", "odd", "wide"])
def test_padded_and_unaligned(calls, monkeypatch, invariant, where):
    """Rows behind the last request are zeros, or as they were in an output that was given; kernels get rows at 16-byte addresses."""
    q, cache, md, scores = _steps(invariant, monkeypatch)
    used = q.shape[0]
    want = 2 * q
    q = torch.cat([q, torch.full_like(q[:1], float("nan")).expand(3, -1, -1)])
    T = q.shape[0]
    q = torch.cat([torch.zeros(T, 1, 24, dtype=q.dtype), q], 1).flatten(1)[:, 20:][:, 4:].unflatten(1, (8, 24))      # a slice of wider rows
    out = {"": None, "given": torch.full((T, 8, 24), 7.0, dtype=q.dtype), "odd": torch.full((T * 192 + 4,), 7.0, dtype=q.dtype)[4:].view(T, 8, 24),
           "wide": torch.full((T, 197), 7.0, dtype=q.dtype)[:, 5:].unflatten(1, (8, 24))}[where]
    got = ops.scored_attention(q, cache, md, 0.1, scores, out=out)
    assert [c[0] for c in calls] == ["attention", "weights"]
    for x in calls[0][1:]:
        assert x is not None and x.data_ptr() % 16 == 0 and x.stride(0) % 8 == 0 and x.stride(1) == 24 and x.stride(2) == 1
    assert torch.equal(got[:used], want) and (got[used:] == (0.0 if out is None else 7.0)).all()
    assert out is None or got is out


def test_key_weights_without_offsets(calls, monkeypatch):
    q, cache, md, scores = _steps(False, monkeypatch)
    with pytest.raises(ValueError):
        ops.key_weights(q, cache, dataclasses.replace(md, query_start_loc=None), 0.1, torch.zeros(25, 8), scores)
    assert not calls


def test_groups_of_a_decode_step():
    """Requests of a launch: all of them where their workspace is small, else as many as have room, in groups of about the same size."""
    for B, Hq, rows in ((1, 32, 700), (64, 32, 1344), (512, 32, 1000), (513, 8, 100), (64, 32, 131072), (512, 32, 131072), (3, 256, 10 ** 6), (1100, 8, 2000)):
        tiles = -(-rows // 64)
        n = cu.scored_group(B, Hq, tiles)
        assert 1 <= n <= min(B, 512) and (n == 1 or n * Hq * tiles * 256 <= cu.SCORED_BYTES)
        groups = -(-B // n)
        assert n == 1 or groups * n < B + groups
        assert groups == max(-(-B // 512), 1) or groups == 1 or (n + 1) * Hq * tiles * 256 > cu.SCORED_BYTES or -(-B // (groups - 1)) * Hq * tiles * 256 > cu.SCORED_BYTES
    assert cu.scored_group(64, 32, 21) == 64 and cu.scored_group(512, 32, 16) == 512


def test_decode_without_rows(calls, monkeypatch):
    """Tables or scores with room for no row: outputs of zeros, nothing is launched."""
    q, cache, md, scores = step([0, 0], [1, 1], 4, 2, 24, 16, torch.bfloat16, "cpu")
    for s, t in ((scores[..., :0], md.block_table), (scores, md.block_table[:, :0])):
        out = torch.full_like(q, 7.0)
        assert not ops.scored_attention(q, cache, dataclasses.replace(md, block_table=t), 0.1, s).any()
        assert ops.scored_attention(q, cache, dataclasses.replace(md, block_table=t), 0.1, s, out=out) is out and not out.any()
    assert not calls


def test_clusters_of_a_decode_step(monkeypatch):
    """A cluster per row where the device runs all of them at a time; of four or two CTAs also in two turns."""
    at_a_time = {8: 15, 4: 36, 2: 74}
    monkeypatch.setattr(cu, "_device", lambda: 0)
    monkeypatch.setattr(cu, "scored_clusters", lambda device, G, D, tiles, parts, *a: at_a_time[parts])
    for pairs, tiles, want in ((1, 11, 8), (15, 11, 8), (16, 11, 0), (32, 11, 0), (15, 32, 8), (15, 33, 0), (36, 4, 4), (72, 4, 4), (73, 4, 0), (74, 2, 2), (148, 1, 2), (149, 1, 0)):
        assert cu.scored_parts(pairs, tiles, 8, 128, 148, 1, False, 0) == want, (pairs, tiles)
    at_a_time[8] = 33
    for pairs, want in ((33, 8), (34, 0)):
        assert cu.scored_parts(pairs, 20, 4, 128, 148, 1, False, 0) == want
    for G, D in ((17, 128), (4, 256)):
        assert cu.scored_parts(1, 4, G, D, 148, 0, False, 0) == 0


@pytest.mark.parametrize("invariant", [False, True])
def test_one_row_of_a_wider_one(calls, monkeypatch, invariant):
    """A single row's distance to the next means nothing, but kernels are told one that is a multiple of 16 bytes."""
    monkeypatch.setattr(cu, "_key_weights", lambda *a: calls.append(("weights", a[20])) or 0)
    if invariant:
        monkeypatch.setenv("VLLM_BATCH_INVARIANT", "1")
    q, cache, md, scores = step([33], [1], 8, 2, 24, 16, torch.bfloat16, "cpu")
    md.decode_only = invariant
    q = torch.cat([q.flatten(1), torch.zeros(1, 5, dtype=q.dtype)], 1).expand(3, -1).contiguous()[:, :192].unflatten(1, (8, 24))[:1]
    assert q.is_contiguous() and q.stride(0) == 197
    ops.scored_attention(q, cache, md, 0.1, scores)
    ops.key_weights(q, cache, md, 0.1, torch.zeros(1, 8), scores)
    assert [c[0] for c in calls] == ["attention", "weights", "weights"]
    assert calls[0][1].stride(0) % 8 == 0 and calls[0][2].stride(0) % 8 == 0 and calls[1][1] % 8 == 0 and calls[2][1] % 8 == 0, calls
