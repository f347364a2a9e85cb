"""A key-value cache in 4 bits: calls that its documentation allows, as far as they show without a device."""
import random
import types

import numpy as np
import pytest
import torch

from tests.fp4_oracle import step
from tests.utils import make_llm
from vllm_b200 import envs, ops
from vllm_b200.layers.attention import attention_layers
from vllm_b200.ops import cuda, ref


def _rnd(*shape):
    return torch.randn(shape, dtype=torch.bfloat16)


LAYOUTS = {
    "interleaved": lambda T, H, D: _rnd(T, H, D, 2)[..., 0],  # keys and values of a channel side by side
    "every other column": lambda T, H, D: _rnd(T, 2 * D)[:, ::2][:, None].expand(T, H, D),
    "one column": lambda T, H, D: _rnd(T, 8)[:, :1, None].expand(T, H, D),
    "heads first": lambda T, H, D: _rnd(H, T, D).transpose(0, 1),
    "columns first": lambda T, H, D: _rnd(H, D, T).permute(2, 0, 1),
    "a token for all": lambda T, H, D: _rnd(1, H, D).expand(T, H, D),
    "part of a projection": lambda T, H, D: _rnd(T, (H + 2) * D)[:, D:-D].unflatten(1, (H, D)),
}


@pytest.mark.parametrize("H", [1, 2])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_rows_lie_as_the_kernel_reads_them(layout, H):
    """Row t, at t times the row stride, has the H D values of a token next to each other, inside the memory that it belongs to."""
    T, D = 3, 16
    x = LAYOUTS[layout](T, H, D)
    rows = cuda._fp4_rows(x)
    step = rows.stride(0)
    assert rows.data_ptr() % 16 == 0 and step % 8 == 0
    assert rows.storage_offset() + (T - 1) * step + H * D <= rows.untyped_storage().nbytes() // 2
    assert torch.equal(rows.as_strided((T, H * D), (step, 1)), x.reshape(T, H * D))


def _entry_takes(D, H, G, few, room):
    """Limits of the kernel of single tokens (vb_attention_fp4): query rows of a request and a kv head, blocks of them in its grid, strips of a launch of one request."""
    cols = 8 if few * G <= 8 else 16 if few * G <= 16 or D > 128 else 24
    blocks = H * -(-few * G // cols)
    return few * G <= 4096 and G <= 64 and blocks <= 65535 and blocks * (-(-room // 64) + cuda.FP4_EXTRA) < 1 << 29


def _choice(queries, lens, room, H, G, D, host):
    md = types.SimpleNamespace(num_reqs=len(lens), max_seq_len=max(lens), host_lens=(np.concatenate(([0], np.cumsum(queries))), np.array(lens)) if host else None)
    return cuda._fp4_choice(md, max(queries), G, sum(queries), room, H, D)[0]


@pytest.mark.parametrize("host", [True, False])
@pytest.mark.parametrize("H,G,D,longest,others,each,rows,room", [(40, 1, 128, 1639, 31, 65, 9000, 10000), (32, 1, 128, 2048, 31, 65, 9000, 10000), (32, 4, 128, 512, 63, 17, 4000, 10000),
                                                                  (1024, 1, 128, 1100, 63, 65, 9000, 10000), (64, 1, 128, 1500, 63, 65, 3000, 1 << 23)])
def test_a_long_request_among_many_short_ones(H, G, D, longest, others, each, rows, room, host):
    """Steps whose mean makes the kernel of single tokens the cheapest: its entry takes what the rule gives it."""
    few = _choice([longest] + [each] * others, [rows] * (others + 1), room, H, G, D, host)
    assert min(longest, max(1, 64 // G)) <= few <= longest and _entry_takes(D, H, G, few, room)
    assert (few == longest) == (room == 10000 and H < 1024)                # (what it can take, it still gets)


def test_the_rule_keeps_to_the_kernels_limits():
    rng = random.Random(0)
    asked = 0
    for _ in range(5000):
        H, G, D = rng.choice([1, 2, 8, 32, 40, 64, 128, 512, 2000]), rng.choice([1, 2, 4, 8, 16, 64]), rng.choice(cuda.FP4_HEADS)
        longest, B, rows = int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 7)), int(2 ** rng.uniform(0, 15))
        queries = [longest, *(rng.randint(1, longest) for _ in range(B - 1))]
        room = max(rows, int(2 ** rng.uniform(10, 20)))
        few = _choice(queries, [max(rows, n) for n in queries], room, H, G, D, rng.random() < 0.5)
        asked += few > max(1, 64 // G)
        assert _entry_takes(D, H, G, few, room), (queries, H, G, D, few)
    assert asked > 100                                   # (of steps that all take it)


def test_decode_steps_in_batch_invariant_mode_are_not_captured(monkeypatch):
    """They go through 16-bit pages, whose number depends on lengths that a captured step does not know."""
    assert ops.fp4_decode_supported(128, 8, torch.bfloat16)
    monkeypatch.setenv("VLLM_BATCH_INVARIANT", "1")
    envs._cache.clear()
    assert cuda.batch_invariant() and not ops.fp4_decode_supported(128, 8, torch.bfloat16)
    monkeypatch.undo()
    envs._cache.clear()
    assert ops.fp4_decode_supported(128, 8, torch.bfloat16)


@pytest.mark.parametrize("axes", [False, True])
def test_positions_outside_the_table(axes, device="cpu", dtype=torch.float32, rots=(16, 24)):
    """They take its first or last row, whether the rotation is the kernel's (multiples of 16) or not."""
    T, Hq, H, D, far = 4, 4, 2, 32, 9
    for rot in rots:
        g = torch.Generator().manual_seed(rot)
        table = torch.randn(far, rot, generator=g).to(device)
        of_pair = (torch.arange(rot // 2, dtype=torch.int32) % 2).to(device)
        got = []
        for positions in ([-3, 0, 8, 50], [0, 0, 8, 8]):
            q, k, v = (torch.randn(T, n * D, generator=torch.Generator().manual_seed(n)).to(dtype).to(device) for n in (Hq, H, H))
            at = torch.tensor(positions, device=device)
            cache = torch.zeros(ops.fp4_cache_shape(1, H, 16, D), dtype=torch.uint8, device=device)
            ops.rope_and_cache_fp4(torch.stack((at, at.flip(0))) if axes else at, q, k, v, table, D, True, cache, torch.arange(T, device=device), axes=of_pair if axes else None)
            got.append((q, cache))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_the_plain_form_takes_the_pages_of_the_step(monkeypatch):
    """Not the whole cache, which would be seven times its bytes in 32 bits."""
    q, cache, md = step([5, 40, 0, 33], [1, 3, 0, 33], 4, 2, 32, 16, torch.float32, "cpu", seed=3, spread=2.0)
    want = ops.paged_attention_fp4(q, cache, md, 0.2)
    many = torch.full((1000, *cache.shape[1:]), 127, dtype=torch.uint8)
    places = torch.randperm(1000, generator=torch.Generator().manual_seed(0))[:cache.shape[0]]
    many[places] = cache
    seen, values_of = [], ref.fp4_cache_values
    monkeypatch.setattr(ref, "fp4_cache_values", lambda kv, *a: seen.append(kv.shape[0]) or values_of(kv, *a))
    table = md.block_table.clone()
    md.block_table = places[table.long()].int()
    assert torch.equal(ops.paged_attention_fp4(q, many, md, 0.2), want) and seen == [1 + 3 + 3]
    for b, n in enumerate(md.seq_lens.tolist()):     # what stands behind a request's pages says nothing
        md.block_table[b, -(-n // 16):] = -7
    assert torch.equal(ops.paged_attention_fp4(q, many, md, 0.2), want)
    md.seq_lens.zero_()                              # no pages at all
    assert (ops.paged_attention_fp4(q, many, md, 0.2) == 0).all()


@pytest.mark.parametrize("queries", [[1, 1], [3, 2]])
def test_rows_behind_the_last_token_stay_in_the_plain_form(queries):
    """A bucket's padding is left as it is in a given output, and finite in a new one, as by the kernels."""
    q, cache, md = step([5, 40], queries, 4, 2, 32, 16, torch.float32, "cpu", seed=3)
    T = q.shape[0]
    want = ops.paged_attention_fp4(q, cache, md, 0.2)
    padded = torch.cat((q, torch.full((3, 4, 32), float("nan"))))
    out = torch.full_like(padded, 7.0)
    assert ops.paged_attention_fp4(padded, cache, md, 0.2, out=out) is out and torch.equal(out[:T], want) and (out[T:] == 7.0).all()
    got = ops.paged_attention_fp4(padded, cache, md, 0.2, out_scale=0.5)
    assert torch.equal(got[:T], want * 0.5) and (got[T:] == 0).all()


def test_memory_of_a_step_is_kept_free():
    """Of the budget of a device, for steps over a cache in 4 bits."""
    for kvd in ("auto", "nvfp4"):
        llm = make_llm("qwen3moe-tiny", kv_cache_dtype=kvd, load_format="dummy", max_num_seqs=3, max_model_len=200, max_num_batched_tokens=64)
        runner = llm.llm_engine.engine_core.engine_core.model_executor.worker.runner
        layer = next(iter(attention_layers().values()))
        want = cuda.fp4_step_bytes(64, 3, 200, layer.num_heads, layer.num_kv_heads, layer.head_size) if kvd == "nvfp4" else 0
        assert runner.cache_workspace_bytes() == want and want >= (cuda.FP4_PART_BYTES if want else 0)
        llm.shutdown()
    one = cuda.fp4_step_bytes(1, 1, 64, 1, 1, 128)
    assert one == cuda.FP4_PART_BYTES + (64 << 20)                                                       # a page: below the parts
    assert cuda.fp4_step_bytes(8192, 256, 131072, 32, 8, 128) == (1 << 30) + 8192 * 32 * 520 + (64 << 20)      # many requests: a gigabyte of pages at a time
    assert cuda.fp4_step_bytes(8192, 1, 1 << 20, 32, 8, 128) == (1 << 32) + 8192 * 32 * 520 + (64 << 20)       # a long one: all of its own
