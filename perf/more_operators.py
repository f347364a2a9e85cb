"""Operators of a key-value cache held in 4 bits, for timing them and for comparing their outputs with plain forms.

    store    new keys (rotated by their positions, of one axis or of several) and values are quantised into the cache, and read back
    read     the cached rows of a batch in 16 bits, request after request
    attend   attention over the cache: one new token per request, a few, or prompts

A case is one call for one layer (store: the write, then the read of what it wrote).  A row of the cache, one token's keys or values of one head, is D
values y = x / factor in groups of 16: a scale e = e4m3(max |y| / 6) and codes e2m1(y / e), to nearest, ties to even; it stands for code * e * factor.
The cache is [blocks, 2, kv heads, page, D / 2 + D / 16] bytes, and a page of one head holds the codes of all its rows (low nibble first), then their
scales.  Pages of a request are spread at random over the cache; what lies behind a request's last row belongs to nobody.  Lengths are spread evenly
between two bounds; queries are as peaked as trained ones (scores of standard deviation 2.5), a few channels of the keys are larger than the others.
"""
import math
import types

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _case(name, op, batch, low, high, heads, kv_heads, head=128, page=64, dtype="bf16", query=1, axes=0, neox=True, cap=0.0, sinks=False, window=0, lse=False,
          k_scale=1.0, v_scale=1.0):
    """``low`` to ``high``: rows in the cache; ``query``: new tokens among them; ``axes``: position numbers of a token (0: no rotation)."""
    c = {"op": op, "batch": batch, "low": low, "high": high, "heads": heads, "kv_heads": kv_heads, "head": head, "page": page, "dtype": dtype, "query": query,
         "axes": axes, "neox": neox, "cap": cap, "sinks": sinks, "window": window, "lse": lse, "k_scale": k_scale, "v_scale": v_scale}
    return {"name": name, **c} if name else c


def listed():
    return [
        # a decode step of a busy server: 64 new tokens, each into a page of its own request
        _case("store chat", "store", 64, 700, 1301, 32, 8, axes=1),
        # a long prompt's keys and values
        _case("store prompt", "store", 1, 8000, 8000, 32, 8, query=8000, axes=1),
        # an image's tokens, with positions in time, height and width, behind a short text; no kv head is shared
        _case("store image", "store", 3, 1777, 2005, 12, 12, dtype="fp16", query=1777, axes=3),
        # cached parts of a batch are needed in 16 bits
        _case("read chat", "read", 64, 700, 1301, 32, 8),
        # odd heads, small pages
        _case("read narrow", "read", 7, 301, 2500, 10, 5, head=80, page=16, dtype="fp16", k_scale=0.75, v_scale=1.5),
        # one user waits for the next token of an answer: launches and latency count
        _case("decode question", "attend", 1, 700, 700, 32, 8),
        # a busy server: 64 requests around a thousand tokens each
        _case("decode chat", "attend", 64, 700, 1301, 32, 8),
        # two long documents: the cache's length has to be split
        _case("decode documents", "attend", 2, 90001, 100000, 32, 8),
        # a model with narrow heads, capped scores, sinks and a window, small pages
        _case("decode narrow", "attend", 24, 60, 924, 16, 8, head=64, page=32, dtype="fp16", cap=30.0, sinks=True, window=700, lse=True),
        # five drafted tokens of each request are verified
        _case("drafts", "attend", 16, 3000, 4101, 32, 8, query=5),
        # a portion of 500 tokens behind a long cached part, narrow heads and small pages
        _case("portion", "attend", 2, 9011, 12000, 16, 4, head=64, page=32, dtype="fp16", query=500, lse=True, k_scale=0.75, v_scale=1.5),
        # a long prompt
        _case("prompt", "attend", 1, 8000, 8000, 32, 8, query=8000),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["store", "read", "attend", "attend"])
    kind = dict(head=rng.choice([32, 64, 80, 96, 128, 128, 128, 192, 256]), page=rng.choice([16, 32, 64, 64]), dtype=rng.choice(["bf16", "fp16"]),
                k_scale=rng.choice([1.0, 1.0, 0.75]), v_scale=rng.choice([1.0, 1.0, 1.5]))
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 4, 5, 8, 16])
    batch = _log(rng, 1, 64)
    if op == "store":
        query = max(1, _log(rng, 1, 4000) // batch)
        low = query + rng.choice([0, _log(rng, 1, 2000)])
        return _case(None, op, batch, low, low + rng.randint(0, low // 4), min(heads, 32), kv_heads, query=query, axes=rng.choice([0, 1, 1, 3]),
                     neox=rng.random() < 0.7, **kind)
    if op == "read":
        high = max(2, _log(rng, 40, 60000 // batch))
        return _case(None, op, batch, rng.randint(max(1, high // 2), high), high, heads, kv_heads, **kind)
    kind.update(cap=rng.choice([0.0, 0.0, 0.0, 30.0, 50.0]), sinks=rng.random() < 0.3, lse=rng.random() < 0.3)
    query = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 3000)])
    if query > 8:                # prompts, or portions of them
        batch = max(1, min(batch, 3000 // query))
        low = query + rng.choice([0, _log(rng, 1, max(2, min(20000, 12000000 // query) // batch))])
        return _case(None, op, batch, low, low + rng.randint(0, low // 4), kv_heads * min(heads // kv_heads, 8), kv_heads, query=query,
                     window=rng.choice([0, 0, rng.randint(1, low)]), **kind)
    high = max(query + 2, _log(rng, 40, 100000 // batch))
    low = rng.randint(max(query, high // 2), high)
    return _case(None, op, batch, low, high, heads, kv_heads, query=query, window=rng.choice([0, 0, rng.randint(1, high)]), **kind)


def _lens(case):
    n, low, high = case["batch"], case["low"], case["high"]
    return [high if n == 1 else low + (high - low) * (i * 37 % n) // (n - 1) if math.gcd(37, n) == 1 else low + (high - low) * i // (n - 1) for i in range(n)]


def _start(case):
    """First new token of each request, and their number."""
    return [i * case["query"] for i in range(case["batch"] + 1)]


def _quantise(x, factor):
    """Codes and scales [..., D / 2] and [..., D / 16] of 32-bit values [..., D]."""
    y = (x / torch.full((), factor, device=x.device)).unflatten(-1, (-1, 16))
    top = y.abs().amax(-1)
    e = (top / torch.full((), 6.0, device=x.device)).clamp(max=448.0).to(torch.float8_e4m3fn)
    m = y.abs() / e.float().unsqueeze(-1)
    code = ((m > 0.25).byte() + (m >= 0.75).byte() + (m > 1.25).byte() + (m >= 1.75).byte() + (m > 2.5).byte() + (m >= 3.5).byte() + (m > 5.0).byte()
            + 8 * (y < 0).byte()).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, e.view(torch.uint8)


def _parts(cache, case):
    """Codes and scales of the pages, [blocks, 2, kv heads, page, ...], as views of the cache."""
    D, page = case["head"], case["page"]
    flat = cache.flatten(3)
    return flat[..., :page * D // 2].unflatten(-1, (page, D // 2)), flat[..., page * D // 2:].unflatten(-1, (page, D // 16))


def _values(codes, scales, factor):
    """The 32-bit values that codes and scales stand for."""
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    y = table[code.int()].unflatten(-1, (-1, 16)) * scales.view(torch.float8_e4m3fn).float().unsqueeze(-1)
    return (y * torch.full((), factor, device=codes.device)).flatten(-2)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, B, H, D, page, new = TYPES[case["dtype"]], case["batch"], case["kv_heads"], case["head"], case["page"], case["query"]
    lens, start = _lens(case), _start(case)
    width = -(-max(lens) // page)
    owned = [-(-n // page) for n in lens]
    blocks = sum(owned) + 3
    order = torch.randperm(blocks, generator=g, device="cuda").int()
    table = torch.zeros(B, width, dtype=torch.int32, device="cuda")
    at = torch.arange(width)[None] < torch.tensor(owned)[:, None]
    table[at.cuda()] = order[:sum(owned)]
    seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    spread = torch.ones(2, H, 1, D, device="cuda")                 # a few channels of the keys are larger
    spread[0, :, :, torch.randperm(D, generator=g, device="cuda")[:D // 16]] = 4.0
    cache = torch.empty(blocks, 2, H, page, D // 2 + D // 16, dtype=torch.uint8, device="cuda")
    codes, scales = _parts(cache, case)
    for b in range(0, blocks, 512):                                # what is cached so far
        x = torch.empty(min(512, blocks - b), 2, H, page, D, device="cuda").normal_(generator=g).mul_(spread).to(dtype).float()
        for part, factor in enumerate((case["k_scale"], case["v_scale"])):
            codes[b:b + 512, part], scales[b:b + 512, part] = _quantise(x[:, part], factor)
    # what the engine hands to an attention call
    md = types.SimpleNamespace(
        num_reqs=B, num_actual_tokens=start[-1], max_query_len=new, max_seq_len=max(lens), query_start_loc=torch.tensor(start, dtype=torch.int32, device="cuda"),
        seq_lens=seq_lens, block_table=table, slot_mapping=None, kv_vt=False, decode_only=new == 1, causal=True, flat=False, num_splits=0, workspace=None,
        query_start_loc_cpu=None, seq_lens_cpu=None, cascade=None, latent_plan=None,
        host_lens=(torch.tensor(start, dtype=torch.int32).numpy(), torch.tensor(lens, dtype=torch.int32).numpy()))
    state = {"case": case, "md": md, "cache": cache, "sinks": None}
    q = torch.empty(start[-1], case["heads"], D, dtype=dtype, device="cuda").normal_(0, 2.5, generator=g)
    if case["op"] == "attend":
        state["q"] = (q.float() / spread[0, 0, 0]).to(dtype)
        if case["sinks"]:
            state["sinks"] = torch.empty(case["heads"], dtype=torch.float32, device="cuda").normal_(generator=g)
        return state
    if case["op"] == "read":
        state["cu"] = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
        return state
    # new tokens: a projection's output, whose queries, keys and values lie side by side
    qkv = torch.empty(start[-1], (case["heads"] + 2 * H) * D, dtype=dtype, device="cuda").normal_(generator=g)
    state["q"], state["k"], state["v"] = qkv.split([case["heads"] * D, H * D, H * D], -1)
    state["k"].unflatten(-1, (H, D)).mul_(spread[0, :, 0].to(dtype))
    places = (seq_lens[:, None] - new + torch.arange(new, device="cuda")).long()                # of the new tokens in their request
    md.slot_mapping = (table.long().gather(1, places // page) * page + places % page).flatten()
    state["cu"], state["first"] = md.query_start_loc, (seq_lens - new).int()
    if case["axes"]:
        far = max(lens)
        inv = 1e4 ** (-torch.arange(0, D, 2, device="cuda").double() / D)
        angle = torch.arange(far, device="cuda").double()[:, None] * inv
        state["table"] = torch.cat((angle.cos(), angle.sin()), -1).float()
        state["positions"] = places.flatten()
        if case["axes"] > 1:     # rows and columns of an image, the same frame; each pair of channels turns by one of the three
            side = max(1, math.isqrt(new))
            i = torch.arange(new, device="cuda")
            first = (seq_lens - new).long()[:, None]
            state["positions"] = torch.stack([(first + x).flatten().clamp(max=far - 1) for x in (i * 0, i // side, i % side)])
            state["axes"] = torch.tensor([j * 3 // (D // 2) for j in range(D // 2)], dtype=torch.int32, device="cuda")
        else:
            state["axes"] = None
    return state


def _turn(x, state):
    """x [tokens, heads, D] in 32 bits, turned by its positions."""
    case = state["case"]
    half = case["head"] // 2
    at = state["table"][state["positions"]]                                                # [tokens, D] or [axes, tokens, D]
    if state["axes"] is not None:
        pair = torch.arange(half, device="cuda")
        at = torch.cat((at[state["axes"].long(), :, pair].t(), at[state["axes"].long(), :, half + pair].t()), -1)
    cos, sin = at[:, None, :half], at[:, None, half:]
    a, b = (x[..., :half], x[..., half:]) if case["neox"] else (x[..., 0::2], x[..., 1::2])
    u, v = a * cos - b * sin, b * cos + a * sin
    return torch.cat((u, v), -1) if case["neox"] else torch.stack((u, v), -1).flatten(-2)


def _store(state):
    case, md = state["case"], state["md"]
    H, D, page, dtype = case["kv_heads"], case["head"], case["page"], state["k"].dtype
    k, v = state["k"].unflatten(-1, (H, D)), state["v"].unflatten(-1, (H, D))
    if case["axes"]:
        q = state["q"].unflatten(-1, (case["heads"], D))
        q.copy_(_turn(q.float(), state))
        k = _turn(k.float(), state).to(dtype)
    codes, scales = _parts(state["cache"], case)
    block, row = md.slot_mapping // page, md.slot_mapping % page
    got = []
    for part, (x, factor) in enumerate(((k, case["k_scale"]), (v, case["v_scale"]))):
        codes[block, part, :, row], scales[block, part, :, row] = _quantise(x.float(), factor)
        got.append(_values(codes[block, part, :, row], scales[block, part, :, row], factor).to(dtype))
    return {"q": state["q"], "k": got[0], "v": got[1]}


def _rows(state, part):
    """Keys (0) or values (1) of all requests in 32 bits, [requests, kv heads, rows, D], zeros behind a request's last row."""
    case, md = state["case"], state["md"]
    codes, scales = (x[:, part][md.block_table.long()].transpose(1, 2).flatten(2, 3) for x in _parts(state["cache"], case))
    x = _values(codes, scales, case["v_scale"] if part else case["k_scale"])
    seen = torch.arange(x.shape[2], device="cuda") < md.seq_lens[:, None]
    return x.masked_fill_(~seen[:, None, :, None], 0.0)


def _read(state):
    md = state["md"]
    got = []
    for part in range(2):
        x = _rows(state, part).transpose(1, 2)
        seen = torch.arange(x.shape[1], device="cuda") < md.seq_lens[:, None]
        got.append(x[seen].to(TYPES[state["case"]["dtype"]]))
    return {"k": got[0], "v": got[1]}


def _attend(state):
    case, md, H = state["case"], state["md"], state["case"]["kv_heads"]
    k, v, t = _rows(state, 0), _rows(state, 1), case["query"]
    q = state["q"].unflatten(0, (-1, t)).unflatten(2, (H, -1)).permute(2, 0, 3, 1, 4).flatten(2, 3).float()     # [kv heads, requests, group * new, D]
    key = torch.arange(k.shape[2], device="cuda")
    place = (md.seq_lens[:, None] - t + torch.arange(t, device="cuda"))[..., None]
    hidden = key > place
    if case["window"]:
        hidden |= key <= place - case["window"]
    hidden = hidden[:, None]                                                               # [requests, 1, new, rows]
    out = torch.empty_like(state["q"])
    lse = torch.empty(out.shape[:2], dtype=torch.float32, device="cuda")
    o = out.unflatten(0, (-1, t)).unflatten(2, (H, -1))
    ol = lse.unflatten(0, (-1, t)).unflatten(2, (H, -1))
    for h in range(H):                                                                     # (a kv head at a time: the scores of all take too much room)
        s = (q[h] @ k[:, h].transpose(1, 2)).unflatten(1, (-1, t)) * case["head"] ** -0.5
        if case["cap"]:
            s = case["cap"] * torch.tanh(s / case["cap"])
        s = s.masked_fill_(hidden, -math.inf)
        total = s.logsumexp(-1, keepdim=True)
        if state["sinks"] is not None:
            total = torch.logaddexp(total, state["sinks"].unflatten(0, (H, -1))[h][None, :, None, None])
        w = s.sub_(total).exp_()
        o[:, :, h] = (w.flatten(1, 2) @ v[:, h]).unflatten(1, (-1, t)).transpose(1, 2).to(out.dtype)
        ol[:, :, h] = total[..., 0].transpose(1, 2)
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


def run(state):
    case = state["case"]
    if own:
        from vllm_b200 import ops
        md, cache, H, D = state["md"], state["cache"], case["kv_heads"], case["head"]
        scales = {"k_scale": case["k_scale"], "v_scale": case["v_scale"]}
        if case["op"] == "attend":
            got = ops.paged_attention_fp4(state["q"], cache, md, D ** -0.5, case["window"] or None, case["cap"], sinks=state["sinks"], return_lse=case["lse"], **scales)
            return {"out": got[0], "lse": got[1]} if case["lse"] else {"out": got}
        if case["op"] == "read":
            n, longest, first, dtype = sum(_lens(case)), md.max_seq_len, None, TYPES[case["dtype"]]
        else:
            n, longest, first, dtype = md.num_actual_tokens, case["query"], state["first"], state["k"].dtype
            if case["axes"]:
                ops.rope_and_cache_fp4(state["positions"], state["q"], state["k"], state["v"], state["table"], D, case["neox"], cache, md.slot_mapping,
                                       axes=state["axes"], **scales)
            else:
                ops.reshape_and_cache_fp4(state["k"].unflatten(-1, (H, D)), state["v"].unflatten(-1, (H, D)), cache, md.slot_mapping, **scales)
        k, v = (torch.empty(n, H, D, dtype=dtype, device=cache.device) for _ in range(2))
        ops.gather_cache_fp4(cache, md.block_table, state["cu"], k, v, longest, seq_starts=first, **scales)
        return {"k": k, "v": v} if case["op"] == "read" else {"q": state["q"], "k": k, "v": v}
    return {"store": _store, "read": _read, "attend": _attend}[case["op"]](state)


def _pairs(case):
    """Pairs of a query and a key that it sees."""
    t, w = case["query"], case["window"]
    if not w:
        return sum(t * n - t * (t - 1) // 2 for n in _lens(case))
    return sum(sum(min(w, p + 1) for p in range(n - t, n)) for n in _lens(case))


def work(case):
    lens, D, H, Hq, new = _lens(case), case["head"], case["kv_heads"], case["heads"], case["batch"] * case["query"]
    row = 2 * H * D                      # values of a token's keys and values
    if case["op"] == "store":            # queries turned, keys and values read and written in 4 bits, and in 16 bits what those stand for
        return {"bytes": new * ((Hq * D * 4 if case["axes"] else 0) + row * (2 + 9 / 16 + 2)), "flops": 0.0}
    if case["op"] == "read":
        return {"bytes": sum(lens) * row * (9 / 16 + 2), "flops": 0.0}
    seen = [min(n, case["window"] + case["query"] - 1) if case["window"] else n for n in lens]
    return {"bytes": sum(seen) * row * 9 / 16 + new * Hq * D * 4, "flops": 4.0 * _pairs(case) * Hq * D}


def exact(case, seed):
    s = prepare(case, seed)
    md, lens, start, H, D, page = s["md"], _lens(case), _start(case), case["kv_heads"], case["head"], case["page"]
    G, t = case["heads"] // H, case["query"]
    factors = (case["k_scale"], case["v_scale"])
    magnitude = torch.tensor(MAGNITUDES, dtype=torch.float64, device="cuda")
    # values of the 127 scales: three bits behind the leading one, multiples of 2^-9 below 2^-6
    scale = torch.tensor([(m / 8 + (e > 0)) * 2.0 ** (max(e, 1) - 7) for e in range(16) for m in range(8)][:127], dtype=torch.float64, device="cuda")

    def nearest(x, table):
        """Number of the table's entry next to x >= 0, the even one of two."""
        up = torch.searchsorted(table, x).clamp(1, len(table) - 1)
        low, high = x - table[up - 1], table[up] - x
        return torch.where((low < high) | ((low == high) & (up % 2 == 1)), up - 1, up)

    def rounded(x, factor):
        """What values [..., D] in 64 bits are stored as."""
        y = (x / factor).unflatten(-1, (-1, 16))
        e = scale[nearest(y.abs().amax(-1) / 6, scale)].unsqueeze(-1)
        m = torch.where(e > 0, y.abs() / e, 0.0)
        return (magnitude[nearest(m, magnitude)] * y.sign() * e * factor).flatten(-2)

    def rows(b, h, part):
        """[rows, D] of one request and head in 64 bits."""
        flat = s["cache"][md.block_table[b, :-(-lens[b] // page)].long(), part, h].flatten(1)
        code = flat[:, :page * D // 2].reshape(-1, D // 2)[:lens[b]].int()
        e = scale[flat[:, page * D // 2:].reshape(-1, D // 16)[:lens[b]].long()]
        low, high = (magnitude[x & 7] * (1 - 2 * (x >> 3)) for x in (code & 15, code >> 4))
        return torch.stack((low, high), -1).reshape(-1, D) * e.repeat_interleave(16, 1) * factors[part]

    if case["op"] == "read":
        return {name: torch.cat([torch.stack([rows(b, h, part) for h in range(H)], 1) for b in range(case["batch"])]) for part, name in enumerate("kv")}
    if case["op"] == "store":
        got = {"q": s["q"].double(), "k": s["k"].double(), "v": s["v"].double()}
        if case["axes"]:
            half, axis = D // 2, s["axes"]
            position = s["positions"][None] if axis is None else s["positions"]
            for name, heads in (("q", case["heads"]), ("k", H)):
                x = got[name].unflatten(-1, (heads, D))
                turned = torch.empty_like(x)
                for j in range(half):
                    i = position[0 if axis is None else int(axis[j])]
                    cos, sin = s["table"][i, j].double()[:, None], s["table"][i, half + j].double()[:, None]
                    at = (j, half + j) if case["neox"] else (2 * j, 2 * j + 1)
                    turned[..., at[0]] = x[..., at[0]] * cos - x[..., at[1]] * sin
                    turned[..., at[1]] = x[..., at[1]] * cos + x[..., at[0]] * sin
                got[name] = turned.flatten(1)
            got["k"] = got["k"].to(TYPES[case["dtype"]]).double()
        return {"q": got["q"], **{name: rounded(got[name].unflatten(-1, (H, D)), factors[part]) for part, name in enumerate("kv")}}
    out = torch.zeros(start[-1], case["heads"], D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(start[-1], case["heads"], dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        for h in range(H):
            k, v, heads = rows(b, h, 0), rows(b, h, 1), slice(h * G, (h + 1) * G)
            for r in range(start[b], start[b + 1], 1024):
                end = min(start[b + 1], r + 1024)
                x = s["q"][r:end, heads].double() @ k.t() * D ** -0.5
                x = torch.tanh(x / case["cap"]) * case["cap"] if case["cap"] else x
                place = (n - start[b + 1] + torch.arange(r, end, device="cuda"))[:, None]
                key = torch.arange(n, device="cuda")
                seen = (key <= place) & ((key > place - case["window"]) if case["window"] else (key >= 0))
                x = x.exp() * seen[:, None]
                total = x.sum(-1, keepdim=True)
                if s["sinks"] is not None:
                    total = total + s["sinks"][heads, None].double().exp()
                out[r:end, heads] = x @ v / total
                lse[r:end, heads] = total[..., 0].log()
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
