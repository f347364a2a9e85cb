"""A key-value cache in 4 bits on the device: writing, reading back and attention against 64 bits."""
import math

import pytest
import torch

from tests.fp4_oracle import CODES, SCALES, attend, quantise, step, values
from vllm_b200 import ops
from vllm_b200.ops import cuda_ops, ref

pytestmark = pytest.mark.gpu
LENS = [1, 15, 16, 17, 63, 64, 65, 300, 1030]
HALVES = [torch.bfloat16, torch.float16]


def _cache(blocks, H, BS, D, fill=0):
    return torch.full(ops.fp4_cache_shape(blocks, H, BS, D), fill, dtype=torch.uint8, device="cuda")


def _row(cache, slot, part, h):
    """(codes, scale bytes) of a row, lists of numbers."""
    nb, _, H, BS, row = cache.shape
    D = row * 16 // 9
    flat = cache[slot // BS, part, h].flatten()
    codes = flat[:BS * D // 2].view(BS, -1)[slot % BS].tolist()
    return [c >> s & 15 for c in codes for s in (0, 4)], flat[BS * D // 2:].view(BS, -1)[slot % BS].tolist()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("H,D,BS,scales", [(2, 128, 64, (1.0, 1.0)), (3, 80, 16, (0.75, 1.3)), (1, 16, 16, (1.0, 2.0)), (5, 256, 32, (1.0, 1.0)), (2, 512, 48, (1.0, 1.0))])
def test_write_is_the_definition(dtype, H, D, BS, scales):
    g = torch.Generator().manual_seed(D)
    T, blocks = 11, 4
    x = torch.randn(T, (2 * H + 1) * D, generator=g) * torch.logspace(-4, 2, T)[:, None]
    x[:, : H * D : 7] = 0.25                                     # values that lie on borders of codes, and equal ones
    x[3, :16], x[4, :16] = 0.0, 1e-5
    x = x.to(dtype).cuda()
    k, v = x[:, :H * D].unflatten(1, (H, D)), x[:, H * D:2 * H * D].unflatten(1, (H, D))
    slots = torch.randperm(blocks * BS, generator=g)[:T]
    slots[2], slots[7] = -1, blocks * BS                         # nowhere
    cache = _cache(blocks, H, BS, D, 0x5a)
    ops.reshape_and_cache_fp4(k, v, cache, slots.cuda(), *scales)
    want = torch.full_like(cache, 0x5a).cpu()
    codes, sc = ref.fp4_parts(want)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < blocks * BS:
            for part, rows in enumerate((k, v)):
                for h in range(H):
                    c, e = quantise(rows[t, h].tolist(), scales[part])
                    codes[s // BS, part, h, s % BS] = torch.tensor([a | b << 4 for a, b in zip(c[::2], c[1::2])], dtype=torch.uint8)
                    sc[s // BS, part, h, s % BS] = torch.tensor(e, dtype=torch.uint8)
    assert torch.equal(cache.cpu(), want)


def test_write_of_borders_and_extremes():
    """Every border between two codes at every scale, infinities, NaN, values above the largest and below the smallest."""
    rows = []
    for e in range(1, 127):
        s = float(SCALES[e])
        rows.append([6 * s, *(m * s for m in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0)), 0.0])
    rows += [[math.inf, 1.0, -math.inf] + [100.0] * 13, [math.nan] + [1.0] * 15, [1.0] * 15 + [math.nan], [60000.0, -3000.0] + [1.0] * 14, [2.0 ** -9] * 16,
             [2.0 ** -20, -(2.0 ** -14)] * 8, [6 * 2.0 ** -10, 2.0 ** -12] * 8, [math.inf, math.nan] * 8]
    x = torch.tensor(rows, dtype=torch.float32).to(torch.float16).cuda()
    T = x.shape[0]
    cache = _cache(-(-T // 16), 1, 16, 16)
    ops.reshape_and_cache_fp4(x[:, None], -x[:, None], cache, torch.arange(T, device="cuda"))
    on_cpu = torch.zeros_like(cache, device="cpu")
    ref.reshape_and_cache_fp4(x[:, None].cpu(), -x[:, None].cpu(), on_cpu, torch.arange(T))
    got, plain = values(cache), values(on_cpu)
    for t in range(T):
        for part in range(2):
            sign = 1 - 2 * part
            codes, scales = quantise([sign * u for u in x[t].tolist()])
            want = CODES[torch.tensor(codes)] * SCALES[scales[0]]
            for have in (got, plain):
                assert torch.equal(have[t // 16, part, 0, t % 16].nan_to_num(1e9), want.nan_to_num(1e9)), (t, part)
    k = torch.empty(T, 1, 16, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    ops.gather_cache_fp4(cache, torch.arange(cache.shape[0], dtype=torch.int32, device="cuda")[None], torch.tensor([0, T], dtype=torch.int32, device="cuda"), k, v, T)
    assert torch.equal(k[:, 0].double().cpu().nan_to_num(1e9), got[:, 0, 0].reshape(-1, 16)[:T].nan_to_num(1e9))      # exact in 16 bits


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("D,rot,neox,axes", [(128, 128, True, 0), (128, 64, True, 0), (64, 64, False, 0), (80, 80, True, 3), (128, 128, True, 3), (96, 32, False, 2),
                                             (80, 40, True, 0), (256, 256, True, 0), (64, 24, False, 3)])
def test_rotation_and_write(dtype, D, rot, neox, axes):
    g = torch.Generator().manual_seed(D + rot)
    T, Hq, H, BS, far = 9, 6, 2, 32, 5000
    qkv = torch.randn(T, (Hq + 2 * H) * D, generator=g).to(dtype).cuda()
    q, k, v = qkv.split([Hq * D, H * D, H * D], -1)
    angle = torch.randn(far, rot // 2, generator=g, dtype=torch.float64) * 10
    table = torch.cat((angle.cos(), angle.sin()), -1).float().cuda()
    positions = torch.randint(0, far, (max(axes, 1), T), generator=g)
    of_pair = torch.randint(0, axes, (rot // 2,), generator=g, dtype=torch.int32) if axes else torch.zeros(rot // 2, dtype=torch.int32)
    slots = torch.randperm(4 * BS, generator=g)[:T]
    cache, before = _cache(4, H, BS, D), qkv.clone()
    got = ops.rope_and_cache_fp4(positions.cuda() if axes else positions[0].cuda(), q, k, v, table, D, neox, cache, slots.cuda(), axes=of_pair.cuda() if axes else None)
    assert got.data_ptr() == q.data_ptr() and torch.equal(qkv[:, Hq * D:], before[:, Hq * D:])                          # k and v as they were
    half, pair = rot // 2, torch.arange(rot // 2)
    at = table.double().cpu()[positions]                                                                                # [axes, T, rot]
    cos, sin = at[of_pair.long(), :, pair].t()[:, None], at[of_pair.long(), :, half + pair].t()[:, None]
    out = []
    for x, heads in ((before[:, :Hq * D], Hq), (before[:, Hq * D:(Hq + H) * D], H)):
        x = x.double().cpu().unflatten(1, (heads, D))
        a, b = (x[..., :half], x[..., half:rot]) if neox else (x[..., :rot:2], x[..., 1:rot:2])
        y, size = x.clone(), torch.zeros_like(x)
        u, w, big = a * cos - b * sin, b * cos + a * sin, (a * cos).abs() + (b * sin).abs() + (b * cos).abs() + (a * sin).abs()
        for part, val in ((y, (u, w)), (size, (big, big))):
            if neox:
                part[..., :half], part[..., half:rot] = val
            else:
                part[..., :rot:2], part[..., 1:rot:2] = val
        out.append((y, size))
    # products and their sum in 32 bits, each rounded, then the type
    step_of = torch.finfo(dtype).eps / 2
    err = (q.double().cpu().unflatten(1, (Hq, D)) - out[0][0]).abs()
    assert (err <= step_of * out[0][0].abs() + 2.0 ** -22 * out[0][1] + 2.0 ** -25).all()
    # the rotation of k is the same arithmetic: it is that of a plain form whose 32-bit steps are rounded one by one, and so are the codes
    x = before[:, Hq * D:(Hq + H) * D].float().unflatten(1, (H, D))
    c32, s32 = (t.float().cuda() for t in (cos, sin))
    a, b = (x[..., :half], x[..., half:rot]) if neox else (x[..., :rot:2], x[..., 1:rot:2])
    u, w = a * c32 - b * s32, b * c32 + a * s32
    y = x.clone()
    if neox:
        y[..., :half], y[..., half:rot] = u, w
    else:
        y[..., :rot:2], y[..., 1:rot:2] = u, w
    want = _cache(4, H, BS, D)
    ops.reshape_and_cache_fp4(y.to(dtype), before[:, (Hq + H) * D:].unflatten(1, (H, D)), want, slots.cuda())
    if rot % 16 == 0:                    # (other rotations are the general op's)
        assert torch.equal(cache, want)
    else:
        assert (values(cache)[:, 1] == values(want)[:, 1]).all() and (values(cache)[:, 0] != values(want)[:, 0]).double().mean() < 0.02


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("H,D,BS", [(2, 128, 64), (3, 80, 16), (1, 16, 32), (2, 256, 48), (4, 32, 128)])
def test_read_back(dtype, H, D, BS):
    lens, scales = [0, 1, 17, 64, 130], (0.75, 1.5)
    _, cache, md = step(lens, [0] * 5, H, H, D, BS, dtype, "cuda", seed=D)
    first, count = [0, 0, 5, 0, 128], [0, 1, 12, 64, 2]
    cu = torch.tensor([0, *torch.tensor(count).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    wide = torch.full((sum(count), 2 * H * D + 8), 7.0, dtype=dtype, device="cuda")
    k, v = wide[:, :H * D].unflatten(1, (H, D)), wide[:, H * D:2 * H * D].unflatten(1, (H, D))
    ops.gather_cache_fp4(cache, md.block_table, cu, k, v, max(count), torch.tensor(first, dtype=torch.int32, device="cuda"), *scales)
    x, at, table = values(cache), 0, md.block_table.tolist()
    f32 = torch.tensor(scales, dtype=torch.float32).double()
    for b in range(5):
        for r in range(first[b], first[b] + count[b]):
            for part, rows in enumerate((k, v)):
                want = (x[table[b][r // BS], part, :, r % BS] * f32[part]).float().to(dtype)
                assert torch.equal(rows[at].cpu(), want), (b, r, part)
            at += 1
    assert (wide[:, 2 * H * D:] == 7.0).all()
    # rows without a page are zeros, a request without rows writes none
    far = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    k, v = (torch.full((3, H, D), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    ops.gather_cache_fp4(cache, md.block_table, far, k, v, 3, torch.tensor([md.block_table.shape[1] * BS - 1], dtype=torch.int32, device="cuda"))
    assert (k[1:] == 0).all() and (v[1:] == 0).all()


def _check(q, cache, md, window=None, cap=0.0, sinks=None, k_scale=1.0, v_scale=1.0, pages=False, spread=None, **kw):
    T, Hq, D = q.shape
    scale = D ** -0.5
    want, norm, mass, terms, big = attend(q, cache, md, scale, window, cap, sinks, (k_scale, v_scale), **{{"alibi_slopes": "alibi", "chunk_size": "chunk"}.get(a, a): b for a, b in kw.items()})
    got, lse = ops.paged_attention_fp4(q, cache, md, scale, window, cap, sinks=sinks, k_scale=k_scale, v_scale=v_scale, return_lse=True, **kw)
    u = torch.finfo(q.dtype).eps / 2
    # scores: 32-bit sums of D products (chains of at most D / 8 + 16 additions, which may cut instead of rounding), a factor, a cap and an exponential of 2^-22 each
    eps = (D / 8 + 16) * 2.0 ** -23 * terms + 8 * 2.0 ** -24 * 1.5 * terms + 2.0 ** -21
    # weights: fp16, in two parts where the output is fp16 (a cache read back to pages: in the output's type); their multiples of 2^-32 of the largest; 32-bit sums
    w = u if pages else 2.0 ** -11 if q.dtype is torch.bfloat16 else 2.0 ** -21
    bound = u * want.abs() + (w + 2 * eps + 2.0 ** -13) * mass + max(md.max_seq_len, 1) * 2.0 ** -31 * big + 2.0 ** -25
    got, lse = got.double().cpu(), lse.double().cpu()
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() / bound).max()
    some = norm > -math.inf
    assert torch.equal(lse > -math.inf, some) and ((lse - norm).abs()[some] <= eps + 2.0 ** -20 + 2.0 ** -22 * norm.abs()[some]).all()
    return got


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("Hq,Hkv,D,BS", [(8, 2, 128, 64), (16, 1, 128, 16), (3, 3, 128, 32), (10, 2, 64, 16), (24, 2, 64, 32), (6, 6, 80, 16), (8, 2, 96, 48), (20, 1, 128, 64),
                                         (4, 2, 256, 64), (16, 1, 256, 16), (6, 2, 32, 128), (9, 1, 192, 64), (40, 1, 64, 64), (4, 2, 48, 64)])
def test_decode(dtype, Hq, Hkv, D, BS):
    q, cache, md = step(LENS, [1] * len(LENS), Hq, Hkv, D, BS, dtype, "cuda", seed=Hq + D, spread=2.0)
    _check(q, cache, md, pages=D == 48)
    g = torch.Generator().manual_seed(1)
    sinks = torch.randn(Hq, generator=g).cuda()
    _check(q, cache, md, window=70, cap=20.0, sinks=sinks, k_scale=0.75, v_scale=1.5, pages=D == 48)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("lens", [[5000], [0, 700, 0], [1] * 3, [130] * 40 + [3000], [64] * 700, [0]])
def test_decode_of_few_and_of_many(dtype, lens):
    """Clusters, equal runs, requests without keys, more requests than a launch takes."""
    q, cache, md = step(lens, [1] * len(lens), 8, 2, 64, 16, dtype, "cuda", seed=len(lens), spread=2.0)
    got = _check(q, cache, md, sinks=torch.randn(8).cuda() if len(lens) == 3 else None)
    for b, n in enumerate(lens):
        assert n > 0 or (got[b] == 0).all()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("host", [True, False])
@pytest.mark.parametrize("Hq,Hkv,D,BS", [(8, 2, 128, 64), (6, 2, 64, 32), (5, 1, 96, 16)])
def test_steps_of_drafts_and_prompts(dtype, host, Hq, Hkv, D, BS):
    queries = [1, 3, 0, 5, 40, 2, 130, 1]
    q, cache, md = step([1, 3, 9, 200, 40, 1000, 300, 77], queries, Hq, Hkv, D, BS, dtype, "cuda", seed=D, spread=2.0, host=host)
    _check(q, cache, md, pages=True)
    _check(q, cache, md, window=50, cap=25.0, sinks=torch.randn(Hq).cuda(), v_scale=0.5, pages=True)
    few, fcache, fmd = step([1, 3, 200, 1000, 64], [1, 3, 4, 2, 4], Hq, Hkv, D, BS, dtype, "cuda", seed=D, spread=2.0, host=host)
    _check(few, fcache, fmd)
    _check(few, fcache, fmd, window=3)


@pytest.mark.parametrize("D,kind", [(128, "alibi_slopes"), (64, "alibi_slopes"), (128, "chunk_size"), (64, "chunk_size"), (64, "causal"), (128, "causal")])
def test_other_masks(D, kind):
    for queries in ([1, 1, 1], [1, 30, 9]):
        q, cache, md = step([20, 90, 200], queries, 4, 2, D, 64, torch.bfloat16, "cuda", seed=D, spread=2.0)
        _check(q, cache, md, pages=True, **{kind: {"alibi_slopes": torch.linspace(0.01, 0.2, 4).cuda(), "chunk_size": 32, "causal": False}[kind]})


@pytest.mark.parametrize("dtype", HALVES)
def test_far_apart_scores(dtype):
    """Scores up to some thousands (weights that are all 0 but one), queries next to the ends of their type, of zeros, and a cache of zeros."""
    q, cache, md = step([300, 70, 1030], [1, 1, 1], 8, 2, 128, 64, dtype, "cuda", seed=3, spread=400.0)
    _check(q, cache, md)
    scale = 2.0 ** 110 if dtype is torch.bfloat16 else 100.0
    q, cache, md = step([300, 70, 1030], [1, 1, 1], 8, 2, 128, 64, dtype, "cuda", seed=3)
    q[0] *= scale
    q[1] /= scale
    q[2] = 0
    got = ops.paged_attention_fp4(q, cache, md, 1.0)
    want = attend(q, cache, md, 1.0)[0]
    assert torch.isfinite(got).all() and (got.double().cpu() - want)[1:].abs().max() < 0.05
    cache.zero_()
    assert (ops.paged_attention_fp4(q, cache, md, 1.0) == 0).all()


def test_layouts_of_queries_and_outputs():
    q, cache, md = step([65, 300], [1, 1], 6, 2, 64, 32, torch.bfloat16, "cuda", seed=9)
    want = ops.paged_attention_fp4(q, cache, md, 0.125)
    wide = torch.zeros(2, 1000, dtype=q.dtype, device="cuda")
    wide[:, 3:3 + 384] = q.flatten(1)
    assert torch.equal(ops.paged_attention_fp4(wide[:, 3:387].unflatten(1, (6, 64)), cache, md, 0.125), want)        # rows at odd addresses
    assert torch.equal(ops.paged_attention_fp4(q.transpose(0, 1).contiguous().transpose(0, 1), cache, md, 0.125), want)
    out = torch.full((2, 1000), 7.0, dtype=q.dtype, device="cuda")
    got = ops.paged_attention_fp4(q, cache, md, 0.125, out=out[:, 5:389].unflatten(1, (6, 64)))
    assert torch.equal(got, want) and (out[:, :5] == 7).all() and (out[:, 389:] == 7).all()
    padded = torch.cat((q, torch.full_like(q, float("nan"))))                                                         # rows of a bucket's padding
    got = ops.paged_attention_fp4(padded, cache, md, 0.125)
    assert torch.equal(got[:2], want) and (got[2:] == 0).all()
    table = torch.full((2, 40), -5, dtype=torch.int32, device="cuda")                                                # entries behind a request's pages say nothing
    table[:, :md.block_table.shape[1]] = md.block_table
    md.block_table = table
    assert torch.equal(ops.paged_attention_fp4(q, cache, md, 0.125), want)


def test_run_of_all_in_graphs():
    """Tokens are stored and attended step after step in two captured graphs at once, on other streams, as eagerly."""
    H, Hq, D, BS, B, dtype = 2, 8, 64, 32, 3, torch.bfloat16
    g = torch.Generator().manual_seed(5)
    angle = torch.randn(200, D // 2, generator=g)
    table = torch.cat((angle.cos(), angle.sin()), -1).cuda()

    def fresh():
        pages = torch.arange(B * 6, dtype=torch.int32, device="cuda").view(B, 6)
        _, _, md = step([1] * B, [1] * B, Hq, H, D, BS, dtype, "cuda", host=False)
        md.block_table, md.max_seq_len = pages, 6 * BS
        return dict(cache=_cache(B * 6, H, BS, D), md=md, qkv=torch.zeros(B, (Hq + 2 * H) * D, dtype=dtype, device="cuda"), pos=torch.zeros(B, dtype=torch.int64, device="cuda"),
                    slots=torch.zeros(B, dtype=torch.int64, device="cuda"))

    def body(s):
        q, k, v = s["qkv"].split([Hq * D, H * D, H * D], -1)
        ops.rope_and_cache_fp4(s["pos"], q, k, v, table, D, True, s["cache"], s["slots"])
        return ops.paged_attention_fp4(q.unflatten(1, (Hq, D)), s["cache"], s["md"], D ** -0.5)

    def load(s, i, seed):
        s["qkv"].copy_(torch.randn(s["qkv"].shape, generator=torch.Generator().manual_seed(seed * 1000 + i)).to(dtype))
        s["pos"].fill_(i)
        s["md"].seq_lens.fill_(i + 1)
        s["slots"].copy_(s["md"].block_table[:, i // BS].long() * BS + i % BS)

    runs = [fresh() for _ in range(3)]
    graphs = []
    for s in runs[:2]:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s["slots"].fill_(-1)
            body(s)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s["out"] = body(s)
        graphs.append((graph, torch.cuda.Stream()))
    for i in range(100):
        for (graph, stream), s, seed in zip(graphs, runs, (1, 2)):
            load(s, i, seed)
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
        for (_, stream), s, seed in zip(graphs, runs, (1, 2)):
            torch.cuda.current_stream().wait_stream(stream)
            s.setdefault("all", []).append(s["out"].clone())
    for seed, s in ((1, runs[0]), (2, runs[1])):
        eager = fresh()
        for i in range(100):
            load(eager, i, seed)
            assert torch.equal(body(eager), s["all"][i]), (seed, i)
        assert torch.equal(eager["cache"], s["cache"])


def test_pages_far_into_a_cache():
    """Byte offsets beyond 32 bits."""
    H, D, BS, dtype = 8, 128, 64, torch.bfloat16
    per = 2 * H * BS * (D // 2 + D // 16)
    blocks = (1 << 32) // per + 40
    cache = torch.empty(ops.fp4_cache_shape(blocks, H, BS, D), dtype=torch.uint8, device="cuda")
    q, small, md = step([100, 200], [1, 1], 16, H, D, BS, dtype, "cuda", seed=2)
    far = torch.arange(small.shape[0], device="cuda") + blocks - small.shape[0]
    cache[far] = small
    want = ops.paged_attention_fp4(q, small, md, 0.1)
    kv = [torch.empty(300, H, D, dtype=dtype, device="cuda") for _ in range(4)]
    cu = torch.tensor([0, 100, 300], dtype=torch.int32, device="cuda")
    ops.gather_cache_fp4(small, md.block_table, cu, kv[0], kv[1], 200)
    md.block_table = far[md.block_table.long()].int()
    assert torch.equal(ops.paged_attention_fp4(q, cache, md, 0.1), want)
    ops.gather_cache_fp4(cache, md.block_table, cu, kv[2], kv[3], 200)
    assert torch.equal(kv[0], kv[2]) and torch.equal(kv[1], kv[3])
    slot = torch.tensor([blocks * BS - 1], device="cuda")
    ops.reshape_and_cache_fp4(kv[0][:1], kv[1][:1], cache, slot)
    near = _cache(1, H, BS, D)
    ops.reshape_and_cache_fp4(kv[0][:1], kv[1][:1], near, slot % BS)
    a, b = ref.fp4_parts(cache[-1:]), ref.fp4_parts(near)
    assert all(torch.equal(x[..., BS - 1, :], y[..., BS - 1, :]) for x, y in zip(a, b))


def test_refusals():
    q, cache, md = step([20, 90], [1, 1], 4, 2, 64, 32, torch.bfloat16, "cuda")
    for bad in (q.float(), q[:1], q[:, :3], q[..., :32]):
        with pytest.raises(ValueError):
            ops.paged_attention_fp4(bad, cache, md, 1.0)
    with pytest.raises(ValueError):
        ops.paged_attention_fp4(q, cache.view(torch.int8), md, 1.0)
    with pytest.raises(ValueError):
        ops.paged_attention_fp4(q, cache[:, :, :, :8], md, 1.0)
    md.block_table = md.block_table.long()
    with pytest.raises(ValueError):
        ops.paged_attention_fp4(q, cache, md, 1.0)
    x = torch.zeros(2, 2, 64, device="cuda")
    with pytest.raises(ValueError):
        ops.reshape_and_cache_fp4(x, x, cache, torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        ops.gather_cache_fp4(cache, md.block_table.int(), torch.tensor([0, 2], dtype=torch.int32, device="cuda"), x, x, 2)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("D", [32, 64, 80, 96, 128, 192, 256])
def test_prompts_straight_from_the_cache(dtype, D):
    """The kernel of prompts for every head, whatever the rule would choose: with and without parts of keys, with requests that are not its own."""
    cu = cuda_ops()
    for lens, queries, Hq, Hkv, BS in (([700, 130, 5], [150, 130, 2], 6, 2, 48), ([2100], [40], 5, 1, 64), ([1300, 9], [33, 9], 8, 4, 16)):
        q, cache, md = step(lens, queries, Hq, Hkv, D, BS, dtype, "cuda", seed=D + len(lens), spread=2.0, host=Hq != 5)
        for window, cap, sinks in ((None, 0.0, None), (65, 25.0, torch.randn(Hq).cuda())):
            out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
            cu._fp4_rows_attention(q, cache, md, D ** -0.5, window, cap, out, lse, sinks, 1.0, 8)
            want, norm, mass, terms, big = attend(q, cache, md, D ** -0.5, window, cap, sinks)
            eps, u = (D / 8 + 16) * 2.0 ** -23 * terms + 8 * 2.0 ** -24 * 1.5 * terms + 2.0 ** -21, torch.finfo(dtype).eps / 2
            bound = u * want.abs() + (2.0 ** -11 + 2 * eps + 2.0 ** -13) * mass + max(lens) * 2.0 ** -31 * big + 2.0 ** -25
            mine = torch.cat([torch.full((n,), n > 8) for n in queries])
            assert ((out.double().cpu() - want).abs() <= bound)[mine].all() and ((lse.double().cpu() - norm).abs() <= eps + 2.0 ** -20 + 2.0 ** -22 * norm.abs())[mine].all()
            assert (out.cpu()[~mine] == 7.0).all() and (lse.cpu()[~mine] == 7.0).all()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("Hq,Hkv,D", [(6, 2, 64), (5, 1, 128), (8, 2, 80), (4, 4, 32)])
def test_prompts_through_wider_pages(dtype, Hq, Hkv, D):
    """Heads that the tensor-core kernel does not take become 128 wide, and a power of two for each kv head."""
    cu = cuda_ops()
    lens, queries = [700, 130, 5, 64], [150, 130, 2, 64]
    q, cache, md = step(lens, queries, Hq, Hkv, D, 32, dtype, "cuda", seed=D, spread=2.0)
    for window, cap, sinks in ((None, 0.0, None), (65, 25.0, torch.randn(Hq).cuda())):
        out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
        cu._fp4_attention_pages(q, cache, md, D ** -0.5, window, cap, True, out, lse, None, sinks, 0, 1.0, 8, True)
        want, norm, mass, terms, big = attend(q, cache, md, D ** -0.5, window, cap, sinks)
        eps, u = (128 / 8 + 16) * 2.0 ** -23 * terms + 8 * 2.0 ** -24 * 1.5 * terms + 2.0 ** -21, torch.finfo(dtype).eps / 2
        bound = u * want.abs() + (u + 2 * eps + 2.0 ** -13) * mass + max(lens) * 2.0 ** -31 * big + 2.0 ** -25
        mine = torch.cat([torch.full((n,), n > 8) for n in queries])
        assert ((out.double().cpu() - want).abs() <= bound)[mine].all() and ((lse.double().cpu() - norm).abs() <= eps + 2.0 ** -20 + 2.0 ** -22 * norm.abs())[mine].all()


def test_prompts_in_more_than_one_go(monkeypatch):
    """A workspace for one request at a time gives what one for all gives, also without lengths on the host."""
    cu = cuda_ops()
    for host in (True, False):
        q, cache, md = step([300, 700, 90, 500], [100, 200, 1, 150], 8, 2, 128, 64, torch.bfloat16, "cuda", seed=1, host=host)
        monkeypatch.setattr(cu, "FP4_PAGES_BYTES", 1 << 30)
        want = ops.paged_attention_fp4(q, cache, md, 0.1, return_lse=True)
        monkeypatch.setattr(cu, "FP4_PAGES_BYTES", 1 << 18)
        got = ops.paged_attention_fp4(q, cache, md, 0.1, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_batch_invariant_rows(monkeypatch):
    """In batch-invariant mode a request's rows do not depend on what else is in the step."""
    monkeypatch.setenv("VLLM_BATCH_INVARIANT", "1")
    q, cache, md = step([300, 700, 90], [1, 1, 1], 8, 2, 128, 64, torch.bfloat16, "cuda", seed=1)
    want = ops.paged_attention_fp4(q, cache, md, 0.1)
    for b in range(3):
        _, _, one = step([300], [1], 8, 2, 128, 64, torch.bfloat16, "cuda")
        one.seq_lens, one.block_table, one.max_seq_len, one.host_lens = md.seq_lens[b:b + 1], md.block_table[b:b + 1], 700, None
        assert torch.equal(ops.paged_attention_fp4(q[b:b + 1], cache, one, 0.1), want[b:b + 1])


def _llm(model, **kw):
    from vllm_b200 import LLM
    from vllm_b200.model_loader import initialize_dummy_weights
    llm = LLM(model, **{**dict(max_model_len=512, max_num_seqs=16, max_num_batched_tokens=512, gpu_memory_utilization=0.2, load_format="dummy",
                               cudagraph_capture_sizes=[1, 2, 4, 8], dtype="bfloat16"), **kw})
    runner = llm.llm_engine.engine_core.engine_core.model_executor.worker.runner
    with torch.no_grad():
        initialize_dummy_weights(runner.model, 7, -0.05, 0.05)
    return llm, runner


def test_generation_with_a_cache_in_4_bits():
    """Teacher-forced log-probabilities stay near those of a 16-bit cache; captured decode steps give what eager ones give."""
    from vllm_b200 import SamplingParams
    prompts = [{"prompt_token_ids": [(7 * i + j) % 4000 + 3 for j in range(90 + 31 * i)]} for i in range(5)]
    tokens, lps = {}, {}
    for name, kw in (("auto", {}), ("nvfp4", {"kv_cache_dtype": "nvfp4"}), ("eager", {"kv_cache_dtype": "nvfp4", "enforce_eager": True})):
        llm, r = _llm("llama-small", max_num_batched_tokens=64, **kw)                   # chunked: prompts read the cache
        outs = llm.generate(prompts, SamplingParams(max_tokens=12, temperature=0.0, ignore_eos=True, prompt_logprobs=0))
        lps[name] = [list(d.values())[0].logprob for o in outs for d in o.prompt_logprobs[1:]]
        tokens[name] = [o.outputs[0].token_ids for o in outs]
        cache = next(iter(r.kv_caches.values()))
        assert (cache.dtype == torch.uint8) == (name != "auto") and bool(r.graphs) == (name != "eager")
        llm.shutdown()
        del r
    assert tokens["nvfp4"] == tokens["eager"]
    d = sorted(abs(a - b) for a, b in zip(lps["auto"], lps["nvfp4"]))
    assert 0 < d[-1] and d[len(d) // 2] < 0.2 and d[int(0.95 * len(d))] < 0.7, d[-5:]


@pytest.mark.parametrize("model", ["gemma2-tiny", "gptoss-tiny", "qwen2vl-tiny", "qwen3moe-tiny", "bloom-tiny"])
def test_families_with_a_cache_in_4_bits(model):
    from vllm_b200 import SamplingParams
    try:
        llm, _ = _llm(model, kv_cache_dtype="nvfp4", max_model_len=256, max_num_batched_tokens=64, block_size=16)
    except ValueError as e:
        assert "4 bits" in str(e)
        return
    outs = llm.generate([{"prompt_token_ids": [5, 7, 11, 13] * n} for n in (3, 30)], SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True, logprobs=0))
    assert all(len(o.outputs[0].token_ids) == 6 and all(math.isfinite(x.logprob) for d in o.outputs[0].logprobs for x in d.values()) for o in outs)
    llm.shutdown()


@pytest.mark.parametrize("queries", [[1, 1, 1], [200, 1, 90]])
def test_rows_behind_the_last_token_stay(queries):
    """A bucket's padding is left as it is in a given output, and finite in a new one, whichever kernels the step takes."""
    for D, Hq in ((64, 6), (128, 8), (256, 4)):
        q, cache, md = step([300, 90, 1000], queries, Hq, 2, D, 32, torch.bfloat16, "cuda", seed=D)
        T = q.shape[0]
        padded = torch.cat((q, torch.full((5, Hq, D), float("nan"), dtype=q.dtype, device="cuda")))
        want = ops.paged_attention_fp4(q, cache, md, 0.1)
        out = torch.full_like(padded, 7.0)
        assert ops.paged_attention_fp4(padded, cache, md, 0.1, out=out) is out and torch.equal(out[:T], want) and (out[T:] == 7.0).all()
        odd = torch.full((T + 5, Hq * D + 3), 7.0, dtype=q.dtype, device="cuda")
        ops.paged_attention_fp4(padded, cache, md, 0.1, out=odd[:, 3:].unflatten(1, (Hq, D)))
        assert torch.equal(odd[:T, 3:].unflatten(1, (Hq, D)), want) and (odd[T:] == 7.0).all() and (odd[:, :3] == 7.0).all()
        got = ops.paged_attention_fp4(padded, cache, md, 0.1)
        assert torch.equal(got[:T], want) and torch.isfinite(got).all()


def test_max_seq_len_is_a_hint_for_single_tokens():
    q, cache, md = step([5000, 64, 700], [1, 1, 1], 8, 2, 128, 64, torch.bfloat16, "cuda", seed=4)
    want = ops.paged_attention_fp4(q, cache, md, 0.1)
    for hint in (1, 100, 100000):
        md.max_seq_len = hint
        got = ops.paged_attention_fp4(q, cache, md, 0.1)
        assert (got.double() - want.double()).abs().max() < 0.02 and (got != 0).any()
    md.block_table = md.block_table[:, :0]                       # tables without pages: requests without keys
    assert (ops.paged_attention_fp4(q, cache, md, 0.1) == 0).all()


@pytest.mark.parametrize("D,queries", [(128, [1, 1]), (64, [1, 1]), (256, [100, 100]), (128, [100, 100])])
def test_nan_comes_out(D, queries):
    """Of a query, and of keys that are seen; other rows stay as they are."""
    q, cache, md = step([300, 200], queries, 4, 2, D, 64, torch.bfloat16, "cuda", seed=4)
    want = ops.paged_attention_fp4(q, cache, md, 0.1)
    q[0, 1] = float("nan")
    got = ops.paged_attention_fp4(q, cache, md, 0.1)
    assert torch.isnan(got[0, 1]).all()
    got[0, 1] = want[0, 1]
    same = torch.ones_like(got, dtype=torch.bool) if queries[0] == 1 else torch.arange(got.shape[0], device="cuda")[:, None, None] >= 100      # (rows of one warp grow together)
    assert torch.equal(got[same.expand_as(got)], want[same.expand_as(got)]) and (got.double() - want.double()).abs().max() < 0.05


def test_many_tables_with_much_room():
    """Numbers of strips beyond 32 bits: several launches."""
    q, cache, md = step([100] * 40, [1] * 40, 8, 8, 64, 16, torch.bfloat16, "cuda", seed=4)
    want = ops.paged_attention_fp4(q, cache, md, 0.1)
    wide = torch.full((40, 10_000_000), -1, dtype=torch.int32, device="cuda")
    wide[:, :md.block_table.shape[1]] = md.block_table
    md.block_table, md.max_seq_len = wide, 160_000_000
    got = ops.paged_attention_fp4(q, cache, md, 0.1)
    assert (got.double() - want.double()).abs().max() < 0.02 and cuda_ops().fp4_schedule(0, 40, 8, 1, 64, 1, 2_500_000, 2_500_000)[4] > 2


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("D,lens,queries,few", [(64, [4500, 9], [24, 9], 0), (192, [4500], [20], 0), (128, [900, 256], [256, 250], 256), (192, [500, 700], [256, 33], 256), (80, [1300], [128], 128)])
def test_most_parts_and_most_rows(dtype, D, lens, queries, few):
    """Prompts in as many parts of keys as there may be (few = 0), and the kernel of single tokens with as many rows as the rule gives it."""
    cu, G = cuda_ops(), 2048 // few if few else 4
    q, cache, md = step(lens, queries, G, 1, D, 32, dtype, "cuda", seed=D, spread=2.0)
    out, lse, scale = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda"), D ** -0.5
    if few:
        cu._fp4_few(q, cache, md, 1, D, 32, md.block_table.shape[1] * 32, scale, None, 0.0, out, lse, None, 1.0, few)
    else:
        cu._fp4_rows_attention(q, cache, md, scale, None, 0.0, out, lse, None, 1.0, few)
    want, norm, mass, terms, big = attend(q, cache, md, scale, None, 0.0, None)
    eps, u = (D / 8 + 16) * 2.0 ** -23 * terms + 8 * 2.0 ** -24 * 1.5 * terms + 2.0 ** -21, torch.finfo(dtype).eps / 2
    bound = u * want.abs() + (2.0 ** -11 + 2 * eps + 2.0 ** -13) * mass + max(lens) * 2.0 ** -31 * big + 2.0 ** -25
    assert ((out.double().cpu() - want).abs() <= bound).all() and ((lse.double().cpu() - norm).abs() <= eps + 2.0 ** -20 + 2.0 ** -22 * norm.abs()).all()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("D", [64, 128, 192])
@pytest.mark.parametrize("lens,queries", [([300, 700, 5, 400, 90], [1, 150, 1, 90, 2]), ([40, 2100, 9], [1, 300, 3]), ([600, 30, 30], [500, 1, 1]), ([3, 7, 130], [1, 1, 130])])
def test_prompts_among_single_tokens(dtype, D, lens, queries):
    """Prompts first, last and in the middle, the kernels' grids over them alone; lengths on the host and not."""
    for host in (True, False):
        q, cache, md = step(lens, queries, 8, 2, D, 32, dtype, "cuda", seed=D, spread=2.0, host=host)
        _check(q, cache, md, pages=D <= 128)
        _check(q, cache, md, window=70, cap=20.0, sinks=torch.linspace(-2, 2, 8).cuda(), pages=D <= 128)


def test_prompts_among_single_tokens_through_pages(monkeypatch):
    """The same with every prompt through 16-bit pages, in one go and in several."""
    cu = cuda_ops()
    monkeypatch.setattr(cu, "fp4_kernels", lambda T, B, longest, rows, H, G, D: (min(longest, max(1, 64 // G)), False))
    for most in (1 << 30, 1 << 19):
        monkeypatch.setattr(cu, "FP4_PAGES_BYTES", most)
        for D in (64, 128):
            q, cache, md = step([300, 700, 5, 400, 90], [1, 150, 1, 90, 2], 6, 2, D, 32, torch.bfloat16, "cuda", seed=D, spread=2.0)
            _check(q, cache, md, pages=True)
