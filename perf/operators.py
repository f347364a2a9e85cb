"""Operators of a key-value cache with a budget, for timing them and for comparing their outputs with plain forms.

    decode   attention of one new token per request over a paged cache, which also adds each key's weights to its score
    weights  the weights that a prompt's queries (all of them or the last ones) give to the cached keys, added to the scores
    evict    the rows of the highest scores stay in the cache, moved to its front

A case is one call for one layer.  The cache has pages [blocks, 2, kv heads, page, head size]; in layout "vt" (heads of 128, pages of 64) the values
of a page are stored transposed.  Pages of a request are spread at random over the cache; what lies behind a request's last row belongs to nobody.
Lengths are spread evenly between two bounds; queries are as peaked as trained ones (scores of standard deviation 2.5), scores so far of the spread
of accumulated weights.  Where an operator works on the state's own buffers, a second pass adds to what the first one left, or moves the same rows again.
"""
import math
import types

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _case(name, op, batch, low, high, heads, kv_heads, head=128, page=64, vt=True, dtype="bf16", query=1, last=0, cap=0.0, sinks=False, keep=0, first=0, recent=0,
          moved=False):
    """``low`` to ``high``: rows in the cache; ``query``: new tokens among them (weights); ``last``: those that count (0: all); ``moved``: an earlier
    eviction has put the rows out of order."""
    c = {"op": op, "batch": batch, "low": low, "high": high, "heads": heads, "kv_heads": kv_heads, "head": head, "page": page, "vt": vt, "dtype": dtype,
         "query": query, "last": last, "cap": cap, "sinks": sinks, "keep": keep, "first": first, "recent": recent, "moved": moved}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one user waits for the next token of an answer: launches and latency count
        _case("decode question", "decode", 1, 700, 700, 32, 8),
        # a busy server: 64 requests around a thousand tokens each
        _case("decode chat", "decode", 64, 700, 1301, 32, 8),
        # two long documents: the cache's length has to be split
        _case("decode documents", "decode", 2, 90001, 100000, 32, 8),
        # a model with narrow heads, capped scores and sinks, small pages
        _case("decode narrow", "decode", 24, 60, 924, 16, 8, head=64, page=32, vt=False, dtype="fp16", cap=30.0, sinks=True),
        # a short prompt, all of whose queries count
        _case("weights question", "weights", 1, 300, 300, 16, 4, query=300),
        # prompts whose last 64 queries choose what stays
        _case("weights window", "weights", 8, 1500, 2101, 32, 8, query=1500, last=64),
        # a long prompt, all queries
        _case("weights prompt", "weights", 1, 8000, 8000, 32, 8, query=8000),
        # a portion of 512 tokens behind a long cached part, narrow heads and small pages
        _case("weights portion", "weights", 2, 20011, 30000, 16, 4, head=64, page=32, vt=False, dtype="fp16", query=512),
        # one user's cache is cut back
        _case("evict question", "evict", 1, 700, 700, 32, 8, keep=512, recent=64),
        # a server cuts back caches that have grown by some hundred rows since the last time
        _case("evict chat", "evict", 64, 1100, 1301, 32, 8, keep=1024, first=4, recent=128, moved=True),
        # long prompts are cut down to a small part before the answer begins
        _case("evict documents", "evict", 4, 28001, 32000, 32, 8, keep=4096, first=4, recent=64),
        # narrow heads, small pages, values as they come
        _case("evict narrow", "evict", 16, 1900, 2101, 16, 4, head=64, page=32, vt=False, dtype="fp16", keep=1500, first=1, recent=33, moved=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["decode", "weights", "evict"])
    vt = rng.random() < 0.6
    head = 128 if vt else rng.choice([64, 80, 96, 128, 256])
    page = 64 if vt else rng.choice([16, 32, 64])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 4, 4, 5, 8, 16])
    kind = dict(head=head, page=page, vt=vt, dtype=rng.choice(["bf16", "fp16"]), cap=rng.choice([0.0, 0.0, 0.0, 30.0, 50.0]))
    batch = _log(rng, 1, 64)
    if op == "decode":
        high = max(2, _log(rng, 40, 100000 // batch))
        return _case(None, op, batch, rng.randint(max(1, high // 2), high), high, kv_heads * group, kv_heads, sinks=rng.random() < 0.3, **kind)
    if op == "weights":
        query = _log(rng, 2, 4000)
        batch = max(1, min(batch, 4000 // query))
        low = query + rng.choice([0, _log(rng, 1, max(2, min(30000, 12000000 // query) // batch))])
        last = rng.choice([0, 0, rng.randint(1, 64)])
        return _case(None, op, batch, low, low + rng.randint(0, low // 4), kv_heads * min(group, 8), kv_heads, query=query, last=last, **kind)
    kind.pop("cap")
    high = max(16, _log(rng, 40, 120000 // batch))
    low = rng.randint(max(1, high // 2), high)
    keep = rng.randint(max(1, low // 8), high)
    first = rng.choice([0, 1, 4])
    first = first if first < keep else 0
    return _case(None, op, batch, low, high, kv_heads * group, kv_heads, keep=keep, first=first, recent=rng.randint(0, (keep - first) // 2), moved=rng.random() < 0.5, **kind)


def _lens(case):
    n, low, high = case["batch"], case["low"], case["high"]
    return [high if n == 1 else low + (high - low) * (i * 37 % n) // (n - 1) if math.gcd(37, n) == 1 else low + (high - low) * i // (n - 1) for i in range(n)]


def _queries(case):
    """New tokens of each request: a longer cache has the longer query."""
    if case["op"] != "weights":
        return [1] * case["batch"]
    return [max(1, case["query"] * n // case["high"]) if case["batch"] > 1 and case["query"] > 1000 else case["query"] for n in _lens(case)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, B, H, D, page = TYPES[case["dtype"]], case["batch"], case["kv_heads"], case["head"], case["page"]
    lens, queries = _lens(case), _queries(case)
    width = -(-max(lens) // page)
    room = (max(lens) // 64 + 1) * 64                      # rows of scores: some for tokens to come
    owned = [-(-n // page) for n in lens]
    blocks = sum(owned) + 3
    order = torch.randperm(blocks, generator=g, device="cuda").int()
    table = torch.zeros(B, width, dtype=torch.int32)
    at = torch.arange(width)[None] < torch.tensor(owned)[:, None]
    table = table.cuda()
    table[at.cuda()] = order[:sum(owned)]
    cache = torch.empty(blocks, 2, H, page, D, dtype=dtype, device="cuda").normal_(generator=g)
    start = [0]
    for n in queries:
        start.append(start[-1] + n)
    q = torch.empty(start[-1], case["heads"], D, dtype=dtype, device="cuda").normal_(0, 2.5, generator=g)
    scores = torch.empty(B, H, room, dtype=torch.float32, device="cuda").exponential_(1.0, generator=g).square_()
    seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    scores *= (torch.arange(room, device="cuda") < seq_lens[:, None, None]) & (case["op"] != "weights" or case["query"] < case["low"])     # a new prompt has none
    # what the engine hands to an attention call
    md = types.SimpleNamespace(
        num_reqs=B, num_actual_tokens=start[-1], max_query_len=max(queries), max_seq_len=max(lens), query_start_loc=torch.tensor(start, dtype=torch.int32, device="cuda"),
        seq_lens=seq_lens, block_table=table, kv_vt=case["vt"], decode_only=case["op"] != "weights", causal=True, flat=False, num_splits=0, workspace=None,
        query_start_loc_cpu=None, seq_lens_cpu=None, cascade=None)
    state = {"case": case, "md": md, "cache": cache, "q": q, "scores": scores, "scale": D ** -0.5, "sinks": None, "positions": None, "lse": None}
    if case["sinks"]:
        state["sinks"] = torch.empty(case["heads"], dtype=torch.float32, device="cuda").normal_(generator=g)
    if case["moved"]:
        # rows as an earlier eviction left them: distinct positions in no order, behind them the tokens since then
        gaps = torch.randint(1, 4, (B, H, room), generator=g, device="cuda")
        old = max(1, min(case["keep"], case["low"] - 1))
        gaps[:, :, old:] = 1
        rows = gaps.cumsum(-1)
        rows = rows - rows[:, :, old - 1:old] + 3 * old
        mixed = torch.rand(B, H, old, generator=g, device="cuda").argsort(-1)
        state["positions"] = torch.cat([rows[:, :, :old].gather(-1, mixed), rows[:, :, old:]], -1).int()
    if case["op"] == "weights":
        # log-sum-exp of every row, as the attention before it returns it: a kv head at a time
        lse = torch.zeros(start[-1], case["heads"], dtype=torch.float32, device="cuda")
        for b in range(B):
            k = _pages(state, 0)[b, :, :lens[b]]
            qb = q[start[b]:start[b + 1]].float().unflatten(1, (H, -1))
            hidden = torch.arange(lens[b], device="cuda") > torch.arange(lens[b] - queries[b], lens[b], device="cuda")[:, None]
            for h in range(H):
                s = _cap(torch.einsum("tgd,nd->tgn", qb[:, h], k[h]) * state["scale"], case["cap"])
                lse[start[b]:start[b + 1]].unflatten(1, (H, -1))[:, h] = s.masked_fill_(hidden[:, None], -math.inf).logsumexp(-1)
            del k
        state["lse"] = lse
    return state


def _cap(s, cap):
    return cap * torch.tanh(s / cap) if cap else s


def _values(cache, vt):
    """The values' part of the cache as [blocks, kv heads, page, head size]."""
    v = cache[:, 1]
    return v.reshape(v.shape[0], v.shape[1], v.shape[3], v.shape[2]).transpose(2, 3) if vt else v


def _pages(state, part, dtype=torch.float32):
    """Keys (0) or values (1) of all requests, [requests, kv heads, rows, head size], zeros behind a request's last row."""
    md, cache = state["md"], state["cache"]
    x = cache[:, 0] if part == 0 else _values(cache, md.kv_vt)
    x = x[md.block_table.long()].transpose(1, 2).flatten(2, 3)
    seen = torch.arange(x.shape[2], device="cuda") < md.seq_lens[:, None]
    return x.to(dtype).masked_fill_(~seen[:, None, :, None], 0.0)


def _decode(state):
    case, md, scores = state["case"], state["md"], state["scores"]
    k, v = _pages(state, 0), _pages(state, 1)
    q = state["q"].float().unflatten(1, (case["kv_heads"], -1))
    s = _cap(q @ k.transpose(2, 3) * state["scale"], case["cap"])                       # [requests, kv heads, group, rows]
    seen = torch.arange(s.shape[-1], device="cuda") < md.seq_lens[:, None, None, None]
    s = s.masked_fill_(~seen, -math.inf)
    lse = s.logsumexp(-1, keepdim=True)
    if state["sinks"] is not None:
        lse = torch.logaddexp(lse, state["sinks"].view(1, case["kv_heads"], -1, 1))
    w = (s - lse).exp_().masked_fill_(~seen, 0.0)
    n = min(s.shape[-1], scores.shape[-1])
    scores[:, :, :n] += w[..., :n].sum(2)
    return {"out": (w @ v).flatten(1, 2).to(state["q"].dtype), "scores": scores}


def _weights(state):
    case, md, scores = state["case"], state["md"], state["scores"]
    k = _pages(state, 0)
    n = min(k.shape[2], scores.shape[-1])
    k = k[:, :, :n]
    begin, end = md.query_start_loc[:-1], md.query_start_loc[1:]
    rows = case["last"] or md.max_query_len
    t = end[:, None] - rows + torch.arange(rows, device="cuda")                            # a request's last rows
    there = t >= begin[:, None]
    t = t.clamp(min=0).long()
    q = state["q"][t].float().unflatten(2, (case["kv_heads"], -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    lse = state["lse"][t].unflatten(2, (case["kv_heads"], -1)).permute(0, 2, 3, 1)
    s = _cap(q @ k.transpose(2, 3) * state["scale"], case["cap"]).unflatten(2, (-1, rows))  # [requests, kv heads, group, query, rows]
    place = md.seq_lens[:, None] - rows + torch.arange(rows, device="cuda")
    seen = (torch.arange(n, device="cuda") <= place[..., None]) & there[..., None]
    w = s.sub_(lse[..., None]).exp_().masked_fill_(~seen[:, None, None], 0.0)
    scores[:, :, :n] += w.sum((2, 3))
    return {"scores": scores}


def _evict(state):
    case, md, scores, cache = state["case"], state["md"], state["scores"], state["cache"]
    rows = torch.arange(scores.shape[-1], device="cuda")
    positions = rows.int().expand(scores.shape) if state["positions"] is None else state["positions"]
    n = md.seq_lens[:, None, None]
    m = n.clamp(max=case["keep"])
    there = rows < n
    total = positions.masked_fill(~there, -1).amax(-1, keepdim=True) + 1
    stays = there & ((positions < case["first"]) | (positions >= total - case["recent"]))
    rank = scores.double().clamp(max=1e300)
    rank = torch.where(rank.isnan() | ~there, -math.inf, rank).masked_fill(stays, math.inf)
    kept = torch.zeros_like(stays).scatter_(-1, rank.sort(dim=-1, descending=True, stable=True)[1], (rows < m).expand(stays.shape))
    b, h, to = (~kept & (rows < m)).nonzero(as_tuple=True)
    source = (kept & (rows >= m)).nonzero(as_tuple=True)[2]                                 # as many of each head, in the same order
    block = lambda r: md.block_table[b, r // case["page"]].long()                          # noqa: E731
    cache[block(to), 0, h, to % case["page"]] = cache[block(source), 0, h, source % case["page"]]
    v = cache[:, 1].view(cache.shape[0], case["kv_heads"], case["head"], case["page"]).transpose(2, 3) if case["vt"] else cache[:, 1]
    v[block(to), h, to % case["page"]] = v[block(source), h, source % case["page"]]
    new = torch.where(rows < m, torch.where(kept, scores, 0.0), 0.0)
    new[b, h, to] = scores[b, h, source]
    places = torch.where(rows < m, positions, total + rows - m).int()
    places[b, h, to] = positions[b, h, source]
    return {"cache": cache, "seq_lens": m.flatten().int(), "scores": new, "positions": places}


def run(state):
    case = state["case"]
    if own:
        from vllm_b200 import ops
        md = state["md"]
        if case["op"] == "decode":
            out = ops.scored_attention(state["q"], state["cache"], md, state["scale"], state["scores"], logits_soft_cap=case["cap"], sinks=state["sinks"])
            return {"out": out, "scores": state["scores"]}
        if case["op"] == "weights":
            ops.key_weights(state["q"], state["cache"], md, state["scale"], state["lse"], state["scores"], logits_soft_cap=case["cap"], last=case["last"])
            return {"scores": state["scores"]}
        seq_lens, scores, positions = ops.evict_keys(state["cache"], md, state["scores"], case["keep"], case["first"], case["recent"], state["positions"])
        return {"cache": state["cache"], "seq_lens": seq_lens, "scores": scores, "positions": positions}
    return {"decode": _decode, "weights": _weights, "evict": _evict}[case["op"]](state)


def work(case):
    lens, D, H, Hq = _lens(case), case["head"], case["kv_heads"], case["heads"]
    rows = sum(lens) * H
    if case["op"] == "decode":           # keys, values, scores read and written, queries and outputs
        return {"bytes": rows * (2 * D * 2 + 8) + case["batch"] * Hq * D * 4, "flops": 4.0 * sum(lens) * Hq * D}
    if case["op"] == "weights":          # keys, scores read and written, queries with their log-sum-exp
        counted = [min(t, case["last"] or t) for t in _queries(case)]
        pairs = sum(t * n - t * (t - 1) // 2 for t, n in zip(counted, lens))
        return {"bytes": rows * (D * 2 + 8) + sum(counted) * Hq * (D * 2 + 4), "flops": 2.0 * pairs * Hq * D}
    # scores and positions read, new ones written; the rows that move, read and written (as many as scores in no order give)
    moves, room = 0.0, (max(lens) // 64 + 1) * 64
    for n in lens:
        m, free = min(n, case["keep"]), n - case["first"] - case["recent"]
        front = m - case["first"] - max(0, m - (n - case["recent"]))
        moves += max(0, front) * (n - m) / max(free, 1)
    return {"bytes": H * (moves * 2 * D * 2 * 2 + sum(lens) * (8 if case["moved"] else 4) + case["batch"] * room * 8), "flops": 0.0}


def exact(case, seed):
    s = prepare(case, seed)
    md, lens, queries, H, cap = s["md"], _lens(case), _queries(case), case["kv_heads"], case["cap"]
    G, page, D = case["heads"] // H, case["page"], case["head"]
    scores, start = s["scores"].double(), md.query_start_loc.tolist()

    def rows(b, h, part):
        """[rows, head size] of one request and head, in 64 bits."""
        got = s["cache"][md.block_table[b, :-(-lens[b] // page)].long(), part, h]
        if part and case["vt"]:
            got = got.reshape(-1, D, page).transpose(1, 2)
        return got.double().reshape(-1, D)[:lens[b]]

    if case["op"] == "evict":
        cache, new, places, left = s["cache"].clone(), torch.zeros_like(scores), torch.zeros_like(scores, dtype=torch.int32), []
        values = cache[:, 1].view(-1, H, D, page) if case["vt"] else cache[:, 1]
        for b, n in enumerate(lens):
            m = min(n, case["keep"])
            left.append(m)
            for h in range(H):
                old = list(range(n)) if s["positions"] is None else s["positions"][b, h, :n].tolist()
                value, total = s["scores"][b, h, :n].tolist(), max(old) + 1
                order = sorted(range(n), key=lambda r: (not (old[r] < case["first"] or old[r] >= total - case["recent"]), -value[r], r))
                stay = set(order[:m])
                holes, sources = [r for r in range(m) if r not in stay], [r for r in range(m, n) if r in stay]
                at = list(range(m))
                for to, source in zip(holes, sources):
                    at[to] = source
                new[b, h, :m] = torch.tensor([value[r] for r in at], dtype=torch.float64, device="cuda")
                places[b, h] = torch.tensor([old[r] for r in at] + [total + i for i in range(scores.shape[-1] - m)], dtype=torch.int32, device="cuda")
                if holes:
                    to, source = torch.tensor(holes, device="cuda"), torch.tensor(sources, device="cuda")
                    tb, sb = md.block_table[b].long()[to // page], md.block_table[b].long()[source // page]
                    cache[tb, 0, h, to % page] = s["cache"][sb, 0, h, source % page]
                    if case["vt"]:
                        values[tb, h, :, to % page] = s["cache"][:, 1].view(-1, H, D, page)[sb, h, :, source % page]
                    else:
                        values[tb, h, to % page] = s["cache"][sb, 1, h, source % page]
        return {"cache": cache.double(), "seq_lens": torch.tensor(left, dtype=torch.int32, device="cuda"), "scores": new, "positions": places}
    out = torch.zeros(case["batch"], case["heads"], D, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        for h in range(H):
            k, heads = rows(b, h, 0), slice(h * G, (h + 1) * G)
            if case["op"] == "decode":
                x = s["q"][b, heads].double() @ k.t() * s["scale"]
                x = (torch.tanh(x / cap) * cap if cap else x).exp()
                total = x.sum(1, keepdim=True)
                if s["sinks"] is not None:
                    total = total + s["sinks"][heads, None].double().exp()
                out[b, heads] = x @ rows(b, h, 1) / total
                scores[b, h, :n] += (x / total).sum(0)
                continue
            t = min(queries[b], case["last"] or queries[b])
            for r in range(0, t, 2048):
                part = range(start[b + 1] - t + r, min(start[b + 1], start[b + 1] - t + r + 2048))
                x = s["q"][part[0]:part[-1] + 1, heads].double() @ k.t() * s["scale"]
                x = (torch.tanh(x / cap) * cap if cap else x) - s["lse"][part[0]:part[-1] + 1, heads, None].double()
                place = n - (start[b + 1] - torch.arange(part[0], part[-1] + 1, device="cuda"))
                seen = torch.arange(n, device="cuda") <= place[:, None]
                scores[b, h, :n] += (x.exp() * seen[:, None]).sum((0, 1))
    return {"out": out, "scores": scores} if case["op"] == "decode" else {"scores": scores}
