"""What the cache operators are measured on: attention of a chunk of new
tokens over the paged KV cache, attention of one new token per row with a
sliding window and sinks, and eviction by accumulated attention weight.

``run`` computes each operator in elementary torch operations (``own`` false)
or through ``soraku_tts_b200.kernels`` (``own`` true); ``exact`` restates the
definition in 64 bits.

Heads are 128 wide, values FP32.  A row has ``cached`` slots filled; its new
tokens take the next slots.  A query at slot i sees slot j <= i when there is
no window, or i - j < window, or j < sinks.
"""

import math

import torch

own = False

HEAD = 128
EPS = 1e-6


def listed():
    return [
        # a few text tokens join both guidance rows of one running utterance (latency counts)
        _case("chunk_cfg_text", "chunk", rows=2, cached=(180, 300), new=(5, 5)),
        # a ragged batch of requests, each with the text of its next sentence
        _case("chunk_ragged_batch", "chunk", rows=16, cached=(97, 1403), new=(1, 96)),
        # whole prompts of a batch: nothing cached yet
        _case("chunk_prompts", "chunk", rows=8, cached=(0, 0), new=(611, 1024)),
        # one piece of a long document's prompt
        _case("chunk_long_prompt", "chunk", rows=1, cached=(8192, 8192), new=(512, 512)),
        # prompt pieces of endless streams: window, sinks, and the weights that eviction goes by
        _case("chunk_window_mass", "chunk", rows=4, cached=(2500, 6001), new=(130, 256), window=1024, sinks=4, mass=True,
              moved=5000),
        # one audio frame of one utterance's two guidance rows (latency counts)
        _case("decode_cfg", "decode", rows=2, cached=(145, 841), window=512, sinks=4),
        # one frame of a full batch of ragged requests
        _case("decode_batch", "decode", rows=128, cached=(120, 842), window=640, sinks=4),
        # endless streams in a bounded window, weights kept
        _case("decode_window_mass", "decode", rows=16, cached=(9000, 16383), window=4096, sinks=16, mass=True, moved=20000),
        # a long cache before it is thinned: everything visible, weights kept
        _case("decode_long_mass", "decode", rows=2, cached=(30001, 32767), mass=True),
        # one utterance's two rows at the length of an ordinary context
        _case("evict_cfg", "evict", rows=2, cached=(746, 842), sinks=4, recent=64, budget=512),
        # a batch of long streams, thinned to a quarter
        _case("evict_batch", "evict", rows=16, cached=(5000, 8192), sinks=16, recent=256, budget=2048),
        # the longest caches
        _case("evict_long", "evict", rows=4, cached=(28000, 32768), sinks=4, recent=1023, budget=8191),
    ]


def _case(name, op, rows, cached, new=(1, 1), window=0, sinks=0, mass=False, moved=0, recent=0, budget=0, heads=16,
          kv_heads=8, page=64):
    return {"name": name, "op": op, "rows": rows, "heads": heads, "kv_heads": kv_heads, "page": page,
            "cached_lo": cached[0], "cached_hi": cached[1], "new_lo": new[0], "new_hi": new[1], "window": window,
            "sinks": sinks, "mass": mass, "moved": moved, "recent": recent, "budget": budget}


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["chunk", "decode", "evict"])
    kv_heads = rng.choice([2, 4, 8, 8])
    heads = kv_heads * rng.choice([1, 2, 2, 3, 4])
    page = rng.choice([16, 64, 64, 128])
    if op == "chunk":
        while True:
            rows, hi, new_hi = _spread(rng, 1, 24), _spread(rng, 1, 8192) - 1, _spread(rng, 1, 1024)
            if rows * new_hi * (hi + new_hi) * heads <= 40_000_000 * 2:
                break
        windowed = rng.random() < 0.5
        return {"op": op, "rows": rows, "heads": heads, "kv_heads": kv_heads, "page": page,
                "cached_lo": int(hi * rng.random()), "cached_hi": hi, "new_lo": _spread(rng, 1, new_hi), "new_hi": new_hi,
                "window": _spread(rng, 1, 4096) if windowed else 0, "sinks": rng.choice([0, 1, 4, 16]) if windowed else 0,
                "mass": rng.random() < 0.5, "moved": rng.choice([0, 0, 7001]), "recent": 0, "budget": 0}
    while True:
        rows, hi = _spread(rng, 1, 200), _spread(rng, 1, 32768)
        if rows * hi <= 131_072:
            break
    if op == "decode":
        windowed = rng.random() < 0.6
        return {"op": op, "rows": rows, "heads": heads, "kv_heads": kv_heads, "page": page,
                "cached_lo": int(hi * rng.random()), "cached_hi": hi, "new_lo": 1, "new_hi": 1,
                "window": _spread(rng, 1, 8192) if windowed else 0, "sinks": rng.choice([0, 1, 4, 33]) if windowed else 0,
                "mass": rng.random() < 0.5, "moved": rng.choice([0, 0, 7001]), "recent": 0, "budget": 0}
    budget = _spread(rng, 1, hi)
    sinks = min(budget, rng.choice([0, 1, 4, 16]))
    return {"op": op, "rows": rows, "heads": heads, "kv_heads": kv_heads, "page": page, "cached_lo": int(hi * rng.random()),
            "cached_hi": hi, "new_lo": 1, "new_hi": 1, "window": 0, "sinks": sinks, "mass": True, "moved": 0,
            "recent": int((budget - sinks) * rng.random()), "budget": budget}


def _lengths(lo, hi, rows):
    # spread over [lo, hi] by the golden ratio, the longest first
    return [hi - int((hi - lo) * ((r * 0.6180339887498949) % 1.0)) for r in range(rows)]


def _sizes(case):
    cached = _lengths(case["cached_lo"], case["cached_hi"], case["rows"])
    new = _lengths(case["new_lo"], case["new_hi"], case["rows"]) if case["op"] != "evict" else [0] * case["rows"]
    return cached, new


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rows, heads, kv_heads, page = case["rows"], case["heads"], case["kv_heads"], case["page"]
    cached, new = _sizes(case)
    need = [-(-(c + n) // page) for c, n in zip(cached, new)]
    pages_row = max(need)
    # the rows' pages lie anywhere in a pool that holds a few more
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32).cpu()
    table = torch.zeros(rows, pages_row, dtype=torch.int32)
    at = 0
    for r in range(rows):
        table[r, :need[r]] = order[at:at + need[r]]
        at += need[r]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    # cached keys are normed heads (root mean square near 1), values are smaller
    pool = normal(n_pages, 2, kv_heads, page, HEAD)
    pool[:, 1] *= 0.4
    s = {"op": case["op"], "n_heads": heads, "n_kv_heads": kv_heads, "page_size": page, "kv_pool": pool,
         "page_table": table.to(dev), "cached": torch.tensor(cached, dtype=torch.int32, device=dev), "window": case["window"],
         "sinks": case["sinks"], "recent": case["recent"], "budget": case["budget"], "mass": None}
    slots = pages_row * page
    if case["mass"] or case["op"] == "evict":
        # long-tailed, as sums of softmax weights are
        s["mass"] = normal(rows, kv_heads, slots).mul_(1.5).exp_()
    if case["op"] != "evict":
        tokens = sum(new)
        start = torch.tensor([0] + new, dtype=torch.int64).cumsum(0).to(torch.int32)
        # `moved`: positions run ahead of the slots once a cache has been thinned
        top = max(c + n for c, n in zip(cached, new)) + case["moved"]
        freq = 1.0 / (1e6 ** (torch.arange(0, HEAD, 2, dtype=torch.float64, device=dev) / HEAD))
        angle = torch.arange(top, dtype=torch.float64, device=dev)[:, None] * freq
        s.update(qkv=normal(tokens, (heads + 2 * kv_heads) * HEAD), q_norm=1 + 0.2 * normal(HEAD), k_norm=1 + 0.2 * normal(HEAD),
                 rope_cos=angle.cos().float(), rope_sin=angle.sin().float(), pos=s["cached"] + case["moved"],
                 chunk_start=start.to(dev), max_chunk=max(new))
    return s


def run(state):
    if state["op"] == "evict":
        return _run_evict(state)
    if own:
        from soraku_tts_b200 import kernels

        keys = ("n_heads", "n_kv_heads", "q_norm", "k_norm", "rope_cos", "rope_sin", "cached", "pos", "kv_pool", "page_table",
                "page_size", "window", "sinks", "mass")
        args = {k: state[k] for k in keys}
        if state["op"] == "chunk":
            out = kernels.chunk_attention(state["qkv"], eps=EPS, chunk_start=state["chunk_start"],
                                          max_chunk=state["max_chunk"], **args)
        else:
            out = kernels.window_decode_attention(state["qkv"], eps=EPS, **args)
    else:
        out = _plain_attention(state)
    return {"out": out, "kv_pool": state["kv_pool"], "mass": state["mass"]}


def _normed(x, weight):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight


def _rotated(x, cos, sin):
    a, b = x[..., :HEAD // 2], x[..., HEAD // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_attention(s):
    H, G, page, pool, table = s["n_heads"], s["n_kv_heads"], s["page_size"], s["kv_pool"], s["page_table"].long()
    rows, rep, dev = table.shape[0], H // G, pool.device
    tokens, most = s["qkv"].shape[0], s["max_chunk"]
    start, cached = s["chunk_start"].long(), s["cached"].long()
    # each token's row, and its place among the row's new tokens
    row = torch.bucketize(torch.arange(tokens, device=dev), start[1:], right=True)
    nth = torch.arange(tokens, device=dev) - start[row]
    place = s["pos"].long()[row] + nth
    cos, sin = s["rope_cos"][place][:, None], s["rope_sin"][place][:, None]
    x = s["qkv"].view(tokens, H + 2 * G, HEAD)
    q = _rotated(_normed(x[:, :H], s["q_norm"]), cos, sin)
    k = _rotated(_normed(x[:, H:H + G], s["k_norm"]), cos, sin)
    slot = cached[row] + nth
    pool[table[row, slot // page], 0, :, slot % page] = k
    pool[table[row, slot // page], 1, :, slot % page] = x[:, H + G:]
    # the slots that any of a row's queries may see: all, or the sinks and the windows' span
    filled = cached + (start[1:] - start[:-1])
    if s["window"] > 0 and s["sinks"] + s["window"] + most < table.shape[1] * page:
        first = torch.clamp(cached - s["window"] + 1, min=s["sinks"])
        seen = torch.cat([torch.arange(s["sinks"], device=dev).expand(rows, -1),
                          first[:, None] + torch.arange(s["window"] + most - 1, device=dev)], 1)
    else:
        seen = torch.arange(table.shape[1] * page, device=dev).expand(rows, -1)
    real = seen < filled[:, None]
    at = torch.where(real, seen, 0)
    pages = torch.gather(table, 1, at // page)
    keys = torch.where(real[:, :, None, None], pool[pages, 0, :, at % page], 0.0).permute(0, 2, 1, 3)
    values = torch.where(real[:, :, None, None], pool[pages, 1, :, at % page], 0.0).permute(0, 2, 1, 3)
    padded = torch.zeros(rows, most, H, HEAD, device=dev)
    padded[row, nth] = q * HEAD ** -0.5
    asked = padded.view(rows, most, G, rep, HEAD).permute(0, 2, 3, 1, 4).reshape(rows, G, rep * most, HEAD)
    scores = (asked @ keys.transpose(2, 3)).view(rows, G, rep, most, -1)
    here = cached[:, None] + torch.arange(most, device=dev)  # a query's own slot
    back = here[:, :, None] - seen[:, None, :]
    visible = real[:, None, :] & (back >= 0) & (here < filled[:, None])[:, :, None]
    if s["window"] > 0:
        visible &= (back < s["window"]) | (seen < s["sinks"])[:, None, :]
    visible = visible[:, None, None]
    scores = torch.where(visible, scores, -torch.inf)
    top = scores.amax(-1, keepdim=True)
    weight = torch.where(visible, torch.exp(scores - torch.where(top > -torch.inf, top, 0.0)), 0.0)
    total = weight.sum(-1, keepdim=True)
    weight = weight / torch.where(total > 0, total, 1.0)
    out = (weight.view(rows, G, rep * most, -1) @ values).view(rows, G, rep, most, HEAD).permute(0, 3, 1, 2, 4)
    if s["mass"] is not None:
        # weights add up over a group's heads and the queries; the new slots begin at nothing
        every = torch.arange(s["mass"].shape[2], device=dev)
        s["mass"].masked_fill_(((every >= cached[:, None]) & (every < filled[:, None]))[:, None], 0.0)
        s["mass"].scatter_add_(2, at[:, None].expand(-1, G, -1), torch.where(real[:, None], weight.sum((2, 3)), 0.0))
    return out.reshape(rows, most, H * HEAD)[row, nth]


def _run_evict(s):
    if own:
        from soraku_tts_b200 import kernels

        kept, mass, cached = kernels.evict_cache(s["mass"], cached=s["cached"], kv_pool=s["kv_pool"], page_table=s["page_table"],
                                                 page_size=s["page_size"], budget=s["budget"], sinks=s["sinks"],
                                                 recent=s["recent"])
    else:
        kept, mass, cached = _plain_evict(s)
    return {"kept": kept, "mass": mass, "cached": cached, "kv_pool": s["kv_pool"]}


def _plain_evict(s):
    page, pool, table, mass, budget = s["page_size"], s["kv_pool"], s["page_table"].long(), s["mass"], s["budget"]
    rows, G, slots = mass.shape
    cached = s["cached"].long()[:, None, None]
    every = torch.arange(slots, device=mass.device).expand(rows, G, -1)
    sure = (every < s["sinks"]) | (every >= cached - s["recent"])
    rank = torch.where(sure, torch.inf, mass)
    rank = torch.where(every < cached, rank, -torch.inf)
    # the first `budget` by weight, ties to the lower slot, then in the order of the slots
    width = min(budget, slots)
    first = torch.sort(rank, dim=2, descending=True, stable=True).indices[:, :, :width]
    real = (torch.arange(width, device=mass.device) < torch.clamp(cached, max=budget)).expand(rows, G, -1)
    kept = torch.where(real, torch.sort(torch.where(real, first, slots), dim=2).values, -1)
    source = torch.where(real, kept, 0)
    r = torch.arange(rows, device=mass.device)[:, None, None].expand_as(source)
    g = torch.arange(G, device=mass.device)[None, :, None].expand_as(source)
    to = torch.arange(width, device=mass.device).expand_as(source)
    moved = pool[table[r, source // page], :, g, source % page]
    pool[table[r, to // page][real], :, g[real], (to % page)[real]] = moved[real]
    left = torch.zeros_like(mass)
    left[:, :, :width] = torch.where(real, torch.gather(mass, 2, source), 0.0)
    whole = torch.full((rows, G, budget), -1, dtype=torch.int32, device=mass.device)
    whole[:, :, :width] = kept.to(torch.int32)
    return whole, left, torch.clamp(s["cached"], max=budget)


def work(case):
    cached, new = _sizes(case)
    H, G = case["heads"], case["kv_heads"]
    if case["op"] == "evict":
        # weights in and out, the slots kept, and each kept row that is not among the first ones to the place of an evicted
        # one; the least that must move is the recent ones and what the weights pick beyond the new end
        nbytes = 0
        for c in cached:
            keep = min(c, case["budget"])
            free = max(0, c - case["sinks"] - case["recent"])
            picked = max(0, keep - case["sinks"] - case["recent"])
            # picks are spread evenly: about one slot in free / picked stays, so nearly all behind the sinks move
            moves = (keep - case["sinks"] if free > picked else 0) if c > keep else 0
            nbytes += G * (4 * c + 8 * keep + max(0, moves) * 2 * 2 * HEAD * 4)
        return {"bytes": nbytes, "flops": 0}
    nbytes = flops = 0
    for c, n in zip(cached, new):
        pairs, first = 0, c
        for i in range(c, c + n):
            if case["window"] > 0:
                low = max(0, i - case["window"] + 1)
                pairs += i + 1 - low + min(case["sinks"], low)
            else:
                pairs += i + 1
        if case["window"] > 0:
            low = max(0, c - case["window"] + 1)
            first = c - low + min(case["sinks"], low)
        # new heads in, outputs out, new keys and values into the cache, visible cached keys and values in
        nbytes += n * (H + 2 * G) * HEAD * 4 + n * H * HEAD * 4 + n * G * 2 * HEAD * 4 + first * G * 2 * HEAD * 4
        nbytes += (2 * first + n) * G * 4 if case["mass"] else 0
        flops += 4 * HEAD * H * pairs
    return {"bytes": nbytes, "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "evict":
        return _exact_evict(s)
    H, G, page = s["n_heads"], s["n_kv_heads"], s["page_size"]
    rep, half = H // G, HEAD // 2
    pool = s["kv_pool"].double()
    mass = None if s["mass"] is None else s["mass"].double()
    table, start, cached, pos = s["page_table"].cpu(), s["chunk_start"].tolist(), s["cached"].tolist(), s["pos"].tolist()
    outs = []
    for r in range(table.shape[0]):
        n, c = start[r + 1] - start[r], cached[r]
        x = s["qkv"][start[r]:start[r + 1]].double().reshape(n, H + 2 * G, HEAD)
        cos, sin = (s[t][pos[r]:pos[r] + n].double() for t in ("rope_cos", "rope_sin"))

        def head(y, w):
            y = w.double() * y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / HEAD + EPS)
            z = torch.empty_like(y)
            z[..., :half] = y[..., :half] * cos[:, None] - y[..., half:] * sin[:, None]
            z[..., half:] = y[..., half:] * cos[:, None] + y[..., :half] * sin[:, None]
            return z

        q, k, v = head(x[:, :H], s["q_norm"]), head(x[:, H:H + G], s["k_norm"]), x[:, H + G:]
        own_pages = [int(p) for p in table[r, :-(-(c + n) // page)]]
        old = pool[own_pages].permute(1, 2, 0, 3, 4).reshape(2, G, -1, HEAD)[:, :, :c]
        # [G, c + n, HEAD]
        K = torch.cat([old[0], k.transpose(0, 1)], 1)
        V = torch.cat([old[1], v.transpose(0, 1)], 1)
        j = torch.arange(c + n, device=pool.device)
        i = torch.arange(c, c + n, device=pool.device)[:, None]
        hidden = j > i
        if s["window"] > 0:
            hidden |= (i - j >= s["window"]) & (j >= s["sinks"])
        out = torch.empty(n, H, HEAD, dtype=torch.float64, device=pool.device)
        if mass is not None:
            mass[r, :, c:c + n] = 0
        for h in range(H):
            score = (q[:, h] @ K[h // rep].T / math.sqrt(HEAD)).masked_fill(hidden, -math.inf)
            w = torch.softmax(score, 1)
            out[:, h] = w @ V[h // rep]
            if mass is not None:
                mass[r, h // rep, :c + n] += w.sum(0)
        for t in range(n):
            pool[own_pages[(c + t) // page], 0, :, (c + t) % page] = k[t]
            pool[own_pages[(c + t) // page], 1, :, (c + t) % page] = v[t]
        outs.append(out.reshape(n, H * HEAD))
    return {"out": torch.cat(outs), "kv_pool": pool, "mass": mass}


def _exact_evict(s):
    page, budget, table = s["page_size"], s["budget"], s["page_table"].cpu()
    pool = s["kv_pool"].double()
    mass = torch.zeros_like(s["mass"], dtype=torch.float64)
    cached = s["cached"].tolist()
    kept = torch.full((mass.shape[0], mass.shape[1], budget), -1, dtype=torch.int32)
    for r, c in enumerate(cached):
        own_pages = [int(p) for p in table[r, :-(-c // page)]]
        for g in range(mass.shape[1]):
            w = s["mass"][r, g, :c].tolist()
            keep = list(range(c))
            if c > budget:
                fixed = list(range(s["sinks"])) + list(range(c - s["recent"], c))
                middle = sorted(range(s["sinks"], c - s["recent"]), key=lambda j: (-w[j], j))
                keep = sorted(fixed + middle[:budget - len(fixed)])
            kept[r, g, :len(keep)] = torch.tensor(keep, dtype=torch.int32)
            here = torch.tensor(keep, device=pool.device)
            flat = pool[own_pages][:, :, g].permute(1, 0, 2, 3).reshape(2, -1, HEAD)
            flat[:, :len(keep)] = flat[:, here].clone()
            pool[own_pages, :, g] = flat.reshape(2, -1, page, HEAD).permute(1, 0, 2, 3)
            mass[r, g, :len(keep)] = s["mass"][r, g][here].double()
    return {"kept": kept, "mass": mass, "cached": torch.tensor([min(c, budget) for c in cached], dtype=torch.int32),
            "kv_pool": pool}
