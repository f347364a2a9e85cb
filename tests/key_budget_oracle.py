"""Scored attention, key weights and eviction in 64 bits, request by request and head by head, and random steps to try them on."""
import torch

from vllm_b200.forward_context import AttentionMetadata


def step(lens, queries, Hq, Hkv, D, BS, dtype, device, vt=False, seed=0, room=0, spread=1.0, spare=2):
    """(q, cache, md, scores): pages in random order, nothing behind the rows but NaN; scores so far of about 1, 0 behind the rows."""
    g = torch.Generator().manual_seed(seed)
    B, width = len(lens), max(1, -(-max(lens) // BS)) + 1
    owned = [-(-n // BS) for n in lens]
    blocks = sum(owned) + spare
    order = torch.randperm(blocks, generator=g)
    table, at = torch.full((B, width), spare and int(order[-1]), dtype=torch.int32), 0
    cache = torch.randn(blocks, 2, Hkv, BS, D, generator=g).to(dtype)
    for b, n in enumerate(owned):
        table[b, :n] = order[at:at + n].int()
        at += n
        if lens[b] % BS:
            cache[int(table[b, n - 1]), :, :, lens[b] % BS:] = float("nan")
    cache[order[at:]] = float("nan")
    start = [0]
    for n in queries:
        start.append(start[-1] + n)
    q = (torch.randn(start[-1], Hq, D, generator=g) * spread).to(dtype)
    room = room or max(lens) + 5
    scores = torch.rand(B, Hkv, room, generator=g) * 2 * (torch.arange(room) < torch.tensor(lens)[:, None, None])
    if vt:
        cache[:, 1] = cache[:, 1].transpose(-1, -2).contiguous().view(blocks, Hkv, BS, D)
    qsl, sl = torch.tensor(start, dtype=torch.int32), torch.tensor(lens, dtype=torch.int32)
    md = AttentionMetadata(num_reqs=B, num_actual_tokens=start[-1], max_query_len=max(queries), max_seq_len=max(lens), query_start_loc=qsl.to(device),
                           seq_lens=sl.to(device), block_table=table.to(device), slot_mapping=torch.empty(0), query_start_loc_cpu=qsl, seq_lens_cpu=sl,
                           decode_only=all(n == 1 for n in queries), kv_vt=vt)
    return q.to(device), cache.to(device), md, scores.to(device)


def rows(cache, md, b, h, n, part):
    """Keys (0) or values (1) of a request's head, [n, D] in 64 bits."""
    BS, D = cache.shape[3:]
    x = cache[md.block_table[b, :-(-n // BS)].long(), part, h]
    if part and md.kv_vt:
        x = x.reshape(-1, D, BS).transpose(1, 2)
    return x.double().reshape(-1, D)[:n]


def attend(q, cache, md, scale, cap=0.0, sinks=None, last=0, lse=None):
    """(output, log-sum-exp, weights that each key gets, sum of weight |value|, largest sum of scale |q_d k_d|); with ``lse`` that one is used."""
    T, Hq, D = q.shape
    H, lens = cache.shape[2], md.seq_lens.tolist()
    start = list(range(len(lens) + 1)) if md.query_start_loc is None else md.query_start_loc.tolist()
    G = Hq // H
    out, mass = (torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device) for _ in range(2))
    norm = torch.full((T, Hq), float("-inf"), dtype=torch.float64, device=q.device)
    weights, terms = torch.zeros(len(lens), H, max(lens), dtype=torch.float64, device=q.device), 0.0
    for b, n in enumerate(lens):
        s, e = start[b], start[b + 1]
        if e == s or n == 0:
            continue
        for h in range(H):
            k, v, x = rows(cache, md, b, h, n, 0), rows(cache, md, b, h, n, 1), q[s:e, h * G:(h + 1) * G].double()
            a = x @ k.t() * scale
            terms = max(terms, float((x.abs() @ k.t().abs()).max() * scale))
            if cap:
                a = cap * torch.tanh(a / cap)
            seen = torch.arange(n, device=q.device) <= torch.arange(n - (e - s), n, device=q.device)[:, None]
            a = a.masked_fill(~seen[:, None], float("-inf"))
            t = torch.logsumexp(a, -1)
            if sinks is not None:
                t = torch.logaddexp(t, sinks[h * G:(h + 1) * G].double())
            norm[s:e, h * G:(h + 1) * G] = t
            if lse is not None:
                t = lse[s:e, h * G:(h + 1) * G].double()
            w = (a - t[..., None]).exp()
            out[s:e, h * G:(h + 1) * G], mass[s:e, h * G:(h + 1) * G] = w @ v, w @ v.abs()
            weights[b, h, :n] = w[max(0, e - s - last) if last else 0:].sum((0, 1))
    return out, norm, weights, mass, terms


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def weight_error(terms, D):
    """Relative error of a weight from 32-bit sums of D products (in chains of at most D / 8 + 16 additions, which may cut instead of rounding:
    2^-23 of the sum of the terms each), a factor, a difference and an exponential of 2^-22, all of scores up to ``terms``."""
    return (D / 8 + 16) * 2.0 ** -23 * terms + 4 * 2.0 ** -24 * 1.5 * terms + 2.0 ** -21


def evict(cache, md, scores, keep, first=0, recent=0, positions=None):
    """(cache, lengths, scores, positions) by sorting lists."""
    B, H, L = scores.shape
    BS, D = cache.shape[3:]
    cache, new, places, lens = cache.clone(), torch.zeros_like(scores), torch.zeros(B, H, L, dtype=torch.int32), []
    values = cache[:, 1].view(-1, H, D, BS).transpose(2, 3) if md.kv_vt else cache[:, 1]
    for b, n in enumerate(md.seq_lens.tolist()):
        m = min(n, keep)
        lens.append(m)
        pages = md.block_table[b].tolist()
        for h in range(H):
            old = list(range(n)) if positions is None else positions[b, h, :n].tolist()
            total = max(old, default=-1) + 1
            value = [float("-inf") if v != v else v for v in scores[b, h, :n].tolist()]
            order = sorted(range(n), key=lambda r: (not (old[r] < first or old[r] >= total - recent), -value[r], r))
            stay = set(order[:m])
            at = list(range(m))
            for to, source in zip([r for r in range(m) if r not in stay], [r for r in range(m, n) if r in stay]):
                at[to] = source
                for x in (cache[:, 0], values):
                    x[pages[to // BS], h, to % BS] = x[pages[source // BS], h, source % BS]
            new[b, h, :m] = scores[b, h, torch.tensor(at, dtype=torch.long, device=scores.device)]
            places[b, h] = torch.tensor([old[r] for r in at] + [total + i for i in range(L - m)], dtype=torch.int32)
    return cache, torch.tensor(lens, dtype=torch.int32), new, places
