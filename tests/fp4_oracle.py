"""A key-value cache in 4 bits in 64 bits, from its definition, and random steps to try it on."""
import math

import torch

from vllm_b200.forward_context import AttentionMetadata

MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
CODES = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), dtype=torch.float64)
# the 127 scales, then NaN; the upper half is not used
SCALES = torch.tensor([(m / 8 + (e > 0)) * 2.0 ** (max(e, 1) - 7) for e in range(16) for m in range(8)][:127] + [math.nan], dtype=torch.float64)


def nearest(x: float, table) -> int:
    """Number of the entry next to x >= 0, the even one of two."""
    best = min(range(len(table)), key=lambda i: (abs(x - table[i]), i % 2))
    return best


def quantise(row, factor=1.0):
    """(codes, scale bytes) of a row, a list of numbers."""
    codes, scales = [], []
    for g in range(0, len(row), 16):
        y = [float(torch.tensor(v, dtype=torch.float32) / torch.tensor(factor, dtype=torch.float32)) for v in row[g:g + 16]]
        if any(v != v for v in y):
            codes += [0] * 16
            scales.append(127)
            continue
        e = nearest(min(max(abs(v) for v in y) / 6, 448.0), SCALES[:127].tolist())
        scales.append(e)
        for v in y:
            code = 0 if e == 0 else nearest(min(abs(v) / float(SCALES[e]), 6.0), MAGNITUDES)
            codes.append(code + 8 * (v < 0 and code > 0))
    return codes, scales


def values(cache, factors=(1.0, 1.0)):
    """[blocks, 2, kv heads, page, D] in 64 bits."""
    nb, _, H, BS, row = cache.shape
    D = row * 16 // 9
    flat = cache.cpu().reshape(nb, 2, H, BS * row)
    codes, scales = flat[..., :BS * D // 2].reshape(nb, 2, H, BS, D // 2).long(), flat[..., BS * D // 2:].reshape(nb, 2, H, BS, D // 16).long()
    x = torch.stack((CODES[codes & 15], CODES[codes >> 4]), -1).flatten(-2) * SCALES[scales].repeat_interleave(16, -1)
    return x * torch.tensor(factors, dtype=torch.float32).double().view(1, 2, 1, 1, 1)


def step(lens, queries, Hq, Hkv, D, BS, dtype, device, seed=0, spread=1.0, host=True):
    """(q, cache, md): codes and scales at random, pages in random order, nothing behind the rows but NaN."""
    g = torch.Generator().manual_seed(seed)
    B, width = len(lens), max(1, -(-max(lens, default=0) // BS)) + 1
    owned = [-(-n // BS) for n in lens]
    blocks = sum(owned) + 2
    order = torch.randperm(blocks, generator=g)
    table, at = torch.full((B, width), int(order[-1]), dtype=torch.int32), 0
    codes = torch.randint(0, 256, (blocks, 2, Hkv, BS, D // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(0x28, 0x34, (blocks, 2, Hkv, BS, D // 16), generator=g, dtype=torch.uint8)      # 0.25 to 0.69: values of about 1
    for b, n in enumerate(owned):
        table[b, :n] = order[at:at + n].int()
        at += n
        if lens[b] % BS:
            scales[int(table[b, n - 1]), :, :, lens[b] % BS:] = 127
    scales[order[at:]] = 127
    cache = torch.cat((codes.flatten(3), scales.flatten(3)), -1).view(blocks, 2, Hkv, BS, D // 2 + D // 16)
    start = [0]
    for n in queries:
        start.append(start[-1] + n)
    q = (torch.randn(start[-1], Hq, D, generator=g) * spread).to(dtype)
    qsl, sl = torch.tensor(start, dtype=torch.int32), torch.tensor(lens, dtype=torch.int32)
    md = AttentionMetadata(num_reqs=B, num_actual_tokens=start[-1], max_query_len=max(queries, default=0), max_seq_len=max(lens, default=0), query_start_loc=qsl.to(device),
                           seq_lens=sl.to(device), block_table=table.to(device), slot_mapping=torch.empty(0), decode_only=all(n == 1 for n in queries))
    if host:
        md.host_lens = (qsl.numpy(), sl.numpy())
    return q.to(device), cache.to(device), md


def attend(q, cache, md, scale, window=None, cap=0.0, sinks=None, factors=(1.0, 1.0), causal=True, alibi=None, chunk=0):
    """(output, log-sum-exp, sum of weight |value|, largest sum of scale |q_d k_d|, largest |value|)."""
    T, Hq, D = q.shape
    H, BS, lens = cache.shape[2], cache.shape[3], md.seq_lens.tolist()
    start, q, x, table = md.query_start_loc.tolist(), q.double().cpu(), values(cache, factors), md.block_table.cpu().long()
    G = Hq // H
    out, mass = (torch.zeros(T, Hq, D, dtype=torch.float64) for _ in range(2))
    norm, terms, big = torch.full((T, Hq), -math.inf, dtype=torch.float64), 0.0, 0.0
    for b, n in enumerate(lens):
        s, e = start[b], start[b + 1]
        if e == s or n == 0:
            if e > s and sinks is not None:
                norm[s:e] = sinks.double().cpu()
            continue
        rows = x[table[b, :-(-n // BS)]].permute(1, 2, 0, 3, 4).reshape(2, H, -1, D)[:, :, :n]
        for h in range(H):
            k, v, heads = rows[0, h], rows[1, h], slice(h * G, (h + 1) * G)
            a = q[s:e, heads] @ k.t() * scale
            terms = max(terms, float((q[s:e, heads].abs() @ k.t().abs()).max() * scale))
            big = max(big, float(v.abs().max()))
            if cap:
                a = cap * torch.tanh(a / cap)
            place, key = torch.arange(n - (e - s), n)[:, None], torch.arange(n)
            if alibi is not None:
                a = a + alibi[heads].double().cpu()[None, :, None] * (key - place)[:, None]
            seen = torch.ones(e - s, n, dtype=torch.bool)
            if causal:
                seen &= key <= place
            if window:
                seen &= key > place - window
                if not causal:
                    seen &= key < place + window
            if chunk:
                seen &= key // chunk == place // chunk
            a = a.masked_fill(~seen[:, None], -math.inf)
            t = torch.logsumexp(a, -1)
            if sinks is not None:
                t = torch.logaddexp(t, sinks[heads].double().cpu())
            norm[s:e, heads] = t
            w = (a - t[..., None]).exp().nan_to_num(0.0)
            out[s:e, heads], mass[s:e, heads] = w @ v, w @ v.abs()
    return out, norm, mass, terms, big
