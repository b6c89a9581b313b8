"""The operators of a serving step around the projections, as cases that can be timed: the plan of a step (page tables, slot
map), the norms and rotation of queries and keys with the store into the paged cache, attention of new tokens over that cache,
and the draw of the next token.

Where `own` is false, `run` computes them with elementary torch operations in 32 bits; where it is true, through
recipe_dev_b200.Context as a host program calls it. Inputs are made on the GPU from the seed alone; lengths follow from the
case, so that a case always is the same amount of work. `exact` gives the same results in 64 bits from the definitions.
"""
import math

import torch

own = False

DEV = "cuda:0"
KV = {"f16": torch.float16, "bf16": torch.bfloat16}
_contexts = {}


def listed():
    llama = dict(q_heads=32, kv_heads=8, head_dim=128)
    return [
        # The plan of a decode step of 64 sequences: one token each, now and then a page.
        dict(name="plan_decode", op="plan", requests=64, cached_lo=1, cached_hi=8191, fresh_lo=1, fresh_hi=1, page=16),
        # The plan of a step that mixes prompts and decoding: 256 sequences, some with nothing new, 32 to 33 thousand tokens.
        dict(name="plan_mixed", op="plan", requests=256, cached_lo=0, cached_hi=4000, fresh_lo=0, fresh_hi=257, page=32),
        # Queries and keys of one decoded token: the smallest call.
        dict(name="rope_one", op="rope", tokens=1, style="pairs", norm=False, rotary=128, page=16, dtype="f16", **llama),
        # 64 sequences decoded together, with a norm for each head, pairs half a head apart.
        dict(name="rope_batch", op="rope", tokens=64, style="halves", norm=True, rotary=128, page=16, dtype="bf16", **llama),
        # A prompt of ragged length.
        dict(name="rope_prompt", op="rope", tokens=2039, style="halves", norm=True, rotary=128, page=16, dtype="f16", **llama),
        # Attention of one decoded token over a short conversation: latency.
        dict(name="attend_one", op="attend", requests=1, cached_lo=1000, cached_hi=1000, fresh_lo=1, fresh_hi=1, page=16, dtype="f16", window=0, **llama),
        # One decoded token at the end of a long document: the cache is read once, by the whole GPU.
        dict(name="attend_long", op="attend", requests=1, cached_lo=131070, cached_hi=131070, fresh_lo=1, fresh_hi=1, page=64, dtype="f16", window=0, **llama),
        # 64 sequences of uneven length decoded together.
        dict(name="attend_batch", op="attend", requests=64, cached_lo=0, cached_hi=8191, fresh_lo=1, fresh_hi=1, page=16, dtype="bf16", window=0, **llama),
        # A chunk of a long prompt: 509 new tokens over what earlier chunks left in the cache.
        dict(name="attend_chunk", op="attend", requests=1, cached_lo=7680, cached_hi=7680, fresh_lo=509, fresh_hi=509, page=16, dtype="f16", window=0, **llama),
        # Whole prompts of uneven length.
        dict(name="attend_prompts", op="attend", requests=4, cached_lo=0, cached_hi=0, fresh_lo=1021, fresh_hi=3001, page=16, dtype="f16", window=0, **llama),
        # The next token of one sequence and of 64, over a large vocabulary.
        dict(name="sample_one", op="sample", rows=1, vocab=262144, top_k=64, top_p=0.95, min_p=0.0, spread=2.5),
        dict(name="sample_batch", op="sample", rows=64, vocab=262144, top_k=0, top_p=0.9, min_p=0.02, spread=2.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "rope", "rope", "attend", "attend", "attend", "attend", "sample", "sample"])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    if op == "plan":
        requests = _log(rng, 1, 512)
        lo = rng.randint(0, 1)
        return dict(op=op, requests=requests, cached_lo=rng.randint(0, 100), cached_hi=_log(rng, 101, 16384), fresh_lo=lo, fresh_hi=max(lo, _log(rng, 1, max(1, 32768 // requests))), page=page)
    heads = dict(rng.choice([dict(q_heads=32, kv_heads=8, head_dim=128), dict(q_heads=32, kv_heads=8, head_dim=128), dict(q_heads=16, kv_heads=16, head_dim=64), dict(q_heads=28, kv_heads=4, head_dim=128),
                             dict(q_heads=8, kv_heads=4, head_dim=256), dict(q_heads=40, kv_heads=2, head_dim=64)]))
    if op == "rope":
        rotary = heads["head_dim"] if rng.random() < 0.75 else heads["head_dim"] // 2
        return dict(op=op, tokens=_log(rng, 1, 4096), style=rng.choice(["halves", "pairs"]), norm=rng.random() < 0.6, rotary=rotary, page=page, dtype=rng.choice(["f16", "bf16"]), **heads)
    if op == "sample":
        rows = _log(rng, 1, 64)
        return dict(op=op, rows=rows, vocab=_log(rng, 1000, 262144), top_k=rng.choice([0, 0, 1, 20, 50, 1000]), top_p=rng.choice([1.0, 0.5, 0.8, 0.95, 0.99]), min_p=rng.choice([0.0, 0.0, 0.01, 0.1]),
                    spread=rng.uniform(1.0, 5.0))
    width = heads["kv_heads"] * heads["head_dim"]
    case = dict(op=op, page=page, dtype=rng.choice(["f16", "bf16"]), window=rng.choice([0, 0, 0, 128, 1000]), **heads)
    if rng.random() < 0.6:  # decoding, sometimes a few tokens a sequence
        requests = _log(rng, 1, 128)
        hi = _log(rng, 16, max(17, min(131070, 100_000_000 // (requests * width))))
        fresh = rng.choice([1, 1, 1, 2, 5])
        return dict(case, requests=requests, cached_lo=rng.randint(0, hi), cached_hi=hi, fresh_lo=1, fresh_hi=fresh)
    requests = rng.choice([1, 1, 2, 3, 6])  # prompts and chunks of prompts
    cached = rng.choice([0, 0, _log(rng, 1, 8192)])
    fresh = _log(rng, 8, 3001)
    while requests * heads["q_heads"] * heads["head_dim"] * fresh * (fresh + cached) > 36_000_000_000:
        cached, fresh = cached // 2, fresh if cached else fresh * 3 // 4
    return dict(case, requests=requests, cached_lo=cached // 2, cached_hi=cached, fresh_lo=max(1, fresh // 3), fresh_hi=fresh)


# ---- inputs --------------------------------------------------------------------------------------------


def _gen(seed, stream):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 64 + stream)


def _spread(lo, hi, n, stride):
    """n whole numbers from lo to hi, evenly, in a mixed order; hi alone for one."""
    while math.gcd(stride, n) != 1:
        stride += 1
    return [hi if n == 1 else lo + (hi - lo) * ((i * stride) % n) // (n - 1) for i in range(n)]


def _lengths(case):
    """Tokens in the cache and new tokens of each request."""
    n = case["requests"]
    return _spread(case["cached_lo"], case["cached_hi"], n, 37), _spread(case["fresh_lo"], case["fresh_hi"], n, 11)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pages(n, page):
    return -(-n // page)


def _rotation(rows, rotary):
    """cos | sin of position * 10000^(-2 i / rotary), as the fp32 table that the rotation reads."""
    angle = torch.arange(rows, dtype=torch.float64, device=DEV)[:, None] * 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=DEV) / rotary)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def prepare(case, seed):
    """The device buffers that a serving loop holds: the batch's lengths, the page table, the cache, activations, logits, and the outputs."""
    s = dict(case=case)
    op = case["op"]
    if op == "plan":
        cached, fresh = _lengths(case)
        page, n = case["page"], case["requests"]
        held = [_pages(c, page) for c in cached]
        need = [_pages(c + f, page) - h for c, f, h in zip(cached, fresh, held)]
        width = max(max(h + w for h, w in zip(held, need)), 1) + 1
        pages = torch.randperm(sum(held) + sum(need) + 8, generator=_gen(seed, 0), device=DEV).int()
        table = torch.full((n, width), -1, dtype=torch.int32, device=DEV)
        mine = torch.arange(width, device=DEV)[None] < torch.tensor(held, device=DEV)[:, None]
        table[mine] = pages[: sum(held)]
        tokens = sum(fresh) + 5  # the arrays of a serving loop are as long as its largest batch
        s |= dict(cached=_int(cached), fresh=_int(fresh), table=table, free=pages[sum(held) :].contiguous(), tokens=tokens)
        s |= dict(starts=torch.empty(n + 1, dtype=torch.int32, device=DEV), lengths=torch.empty(n, dtype=torch.int32, device=DEV), status=torch.empty(3, dtype=torch.int32, device=DEV))
        s |= {k: torch.empty(tokens, dtype=torch.int32, device=DEV) for k in ("slots", "positions", "owners")}
    elif op == "rope":
        t, hq, hk, d, page = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
        gen = _gen(seed, 0)
        qkv = torch.randn((t, (hq + 2 * hk) * d), generator=gen, device=DEV) * torch.exp(0.3 * torch.randn((1, (hq + 2 * hk) * d), generator=gen, device=DEV))
        s["q"], s["k"], s["v"] = qkv[:, : hq * d], qkv[:, hq * d : (hq + hk) * d], qkv[:, (hq + hk) * d :]  # the projections' plane, [q | k | v] a token
        s["q_gain"], s["k_gain"] = (1.0 + 0.2 * torch.randn((2, d), generator=gen, device=DEV)) if case["norm"] else (None, None)
        rows = 8192
        s["rotation"] = _rotation(rows, case["rotary"])
        pages = _pages(t, page) + 3
        perm = torch.randperm(pages, generator=gen, device=DEV)
        at = torch.arange(t, device=DEV)
        s["slots"] = (perm[at // page] * page + at % page).int()
        s["positions"] = (at + torch.randint(0, rows - t, (1,), generator=gen, device=DEV)).int() if t > 256 else torch.randint(0, rows, (t,), generator=gen, device=DEV).int()
        s["k_cache"], s["v_cache"] = (torch.zeros((pages, hk, page, d), dtype=KV[case["dtype"]], device=DEV) for _ in range(2))
        s["q_out"] = torch.empty((t, hq * d), device=DEV)
    elif op == "attend":
        cached, fresh = _lengths(case)
        hq, hk, d, page, n = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], case["requests"]
        gen = _gen(seed, 0)
        held = [_pages(c + f, page) for c, f in zip(cached, fresh)]
        pages, t = sum(held) + 3, sum(fresh)
        s["table"] = torch.full((n, max(held) + 1), -1, dtype=torch.int32, device=DEV)
        mine = torch.arange(max(held) + 1, device=DEV)[None] < torch.tensor(held, device=DEV)[:, None]
        s["table"][mine] = torch.randperm(pages, generator=gen, device=DEV).int()[: sum(held)]
        s["k_cache"], s["v_cache"] = (torch.empty((pages, hk, page, d), dtype=KV[case["dtype"]], device=DEV).normal_(generator=gen) for _ in range(2))
        # some heads look around evenly, some at a few tokens
        s["q"] = torch.randn((t, hq, d), generator=gen, device=DEV) * torch.linspace(0.5, 3.0, hq, device=DEV)[:, None]
        s["starts"], s["lengths"] = _int([sum(fresh[:i]) for i in range(n + 1)]), _int([c + f for c, f in zip(cached, fresh)])
        s["max_fresh"], s["longest"], s["scale"] = max(fresh), max(c + f for c, f in zip(cached, fresh)), d**-0.5
        s["y"] = torch.empty((t, hq, d), device=DEV)
    else:
        rows, vocab = case["rows"], case["vocab"]
        gen = _gen(seed, 0)
        s["logits"] = case["spread"] * torch.randn((rows, vocab), generator=gen, device=DEV)
        s["uniform"] = torch.rand(rows, generator=gen, device=DEV)
        s["temperature"] = 0.6 + 0.6 * torch.rand(rows, generator=gen, device=DEV)
        s["temperature"][7::8] = 0.0  # a few requests of a batch want the best token
        s["top_k"] = torch.full((rows,), case["top_k"], dtype=torch.int32, device=DEV)
        s["top_p"], s["min_p"] = (torch.full((rows,), case[k], device=DEV) for k in ("top_p", "min_p"))
        s["token"], s["kept"] = (torch.empty(rows, dtype=torch.int32, device=DEV) for _ in range(2))
        s["probability"] = torch.empty(rows, device=DEV)
    return s


# ---- one pass ------------------------------------------------------------------------------------------


def _context():
    import recipe_dev_b200 as rq

    if 0 not in _contexts:
        _contexts[0] = rq.Context(0)
    return _contexts[0]


def _cache(s):
    """The cache's handle, kept beside its tensors as a program does."""
    import recipe_dev_b200 as rq

    if "handle" not in s:
        s["handle"] = rq.KvCache(s["k_cache"], s["v_cache"])
    return s["handle"]


def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return {"plan": _plain_plan, "rope": _plain_rope, "attend": _plain_attend, "sample": _plain_sample}[op](s, case)
    ctx = _context()
    if op == "plan":
        ctx.batch_plan(s["cached"], s["fresh"], s["table"], s["free"], case["page"], starts=s["starts"], lengths=s["lengths"], slots=s["slots"], positions=s["positions"], owners=s["owners"], status=s["status"])
        return {k: s[k] for k in ("table", "starts", "lengths", "slots", "positions", "owners", "status")}
    if op == "rope":
        ctx.rope_store(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["rotation"], _cache(s), q_gain=s["q_gain"], k_gain=s["k_gain"], epsilon=1e-6, style=case["style"], q_out=s["q_out"])
        return {k: s[k] for k in ("q_out", "k_cache", "v_cache")}
    if op == "attend":
        return ctx.attention(s["q"], _cache(s), s["table"], s["starts"], s["lengths"], scale=s["scale"], window=case["window"], max_fresh=s["max_fresh"], y=s["y"])
    ctx.sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"], token=s["token"], probability=s["probability"], kept=s["kept"])
    return {k: s[k] for k in ("token", "probability", "kept")}


def _plain_plan(s, case):
    page, tokens = case["page"], s["tokens"]
    cached, fresh, table, free = s["cached"], s["fresh"], s["table"], s["free"]
    held = (cached + page - 1) // page
    need = (cached + fresh + page - 1) // page - held
    before = torch.cumsum(need, 0, dtype=torch.int32) - need
    column = torch.arange(table.shape[1], dtype=torch.int32, device=DEV)[None]
    new = (column >= held[:, None]) & (column < (held + need)[:, None])
    at = before[:, None] + column - held[:, None]
    page_id = torch.where(at < free.numel(), free[at.clamp(0, free.numel() - 1).long()], -1)
    table = torch.where(new, page_id, table)
    ends = torch.cumsum(fresh, 0, dtype=torch.int32)
    starts = torch.cat([ends.new_zeros(1), ends])
    t = torch.arange(tokens, dtype=torch.int32, device=DEV)
    owner = torch.searchsorted(ends, t, right=True, out_int32=True)
    real = owner < fresh.numel()
    r = owner.clamp(max=fresh.numel() - 1).long()
    position = torch.where(real, cached[r] + t - starts[r], 0)
    block = table[r, (position // page).long()]
    slot = torch.where(real & (block >= 0), block * page + position % page, -1)
    total = need.sum(dtype=torch.int32)
    status = torch.stack([ends[-1], total.clamp(max=free.numel()), (total - free.numel()).clamp(min=0)])
    return dict(table=table, starts=starts, lengths=cached + fresh, slots=slot, positions=position, owners=torch.where(real, owner, -1), status=status)


def _plain_rope(s, case):
    t, d, half, page = case["tokens"], case["head_dim"], case["rotary"] // 2, case["page"]
    turn = s["rotation"][s["positions"].long()][:, None]
    cos, sin = turn[..., :half], turn[..., half:]

    def turned(x, gain):
        x = x.reshape(t, -1, d)
        if gain is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gain
        a, b = (x[..., :half], x[..., half : 2 * half]) if case["style"] == "halves" else (x[..., 0 : 2 * half : 2], x[..., 1 : 2 * half : 2])
        a, b = a * cos - b * sin, a * sin + b * cos
        both = torch.cat([a, b], -1) if case["style"] == "halves" else torch.stack([a, b], -1).flatten(-2)
        return torch.cat([both, x[..., 2 * half :]], -1)

    slots = s["slots"].long()
    s["k_cache"][slots // page, :, slots % page] = turned(s["k"], s["k_gain"]).to(s["k_cache"].dtype)
    s["v_cache"][slots // page, :, slots % page] = s["v"].reshape(t, -1, d).to(s["v_cache"].dtype)
    return dict(q_out=turned(s["q"], s["q_gain"]).reshape(t, -1), k_cache=s["k_cache"], v_cache=s["v_cache"])


def _plain_attend(s, case):
    hq, hk, d, page, n = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], case["requests"]
    group, f, longest = hq // hk, s["max_fresh"], s["longest"]
    starts, lengths = s["starts"].long(), s["lengths"].long()
    key = torch.arange(longest, device=DEV)
    block = torch.gather(s["table"].long(), 1, (key // page)[None].expand(n, -1).clamp(max=s["table"].shape[1] - 1)).clamp(min=0)
    k, v = (c[block, :, (key % page)[None]].float().transpose(1, 2) for c in (s["k_cache"], s["v_cache"]))  # [requests, heads, keys, d]
    fresh = starts[1:] - starts[:-1]
    i = torch.arange(f, device=DEV)
    row = (starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][row].reshape(n, f, hk, group, d).permute(0, 2, 1, 3, 4).reshape(n, hk, f * group, d) * s["scale"]
    position = (lengths - fresh)[:, None] + i
    seen = (key <= position[..., None]) & (key < lengths[:, None, None])
    if case["window"]:
        seen = seen & (key > position[..., None] - case["window"])
    seen = seen[:, None].repeat_interleave(group, 2)
    score = torch.where(seen, q @ k.transpose(2, 3), -torch.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -torch.inf, 0.0, top))
    total = weight.sum(-1, keepdim=True)
    y = (weight @ v) / torch.where(total == 0, 1.0, total)
    y = y.reshape(n, hk, f, group, d).permute(0, 2, 1, 3, 4).reshape(n, f, hq, d)
    return y[i[None] < fresh[:, None]]


def _plain_sample(s, case):
    x, t = s["logits"], s["temperature"][:, None]
    top = x.amax(1, keepdim=True)
    scaled = (x - top) / torch.where(t > 0, t, 1.0)
    e = torch.where(t > 0, torch.exp(scaled), (x == top).float())
    mass = (e * 1099511627776.0).long()  # whole numbers of 2^-40: their sums are the same in every order
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    sorted_mass = mass.gather(1, order)
    rank = torch.arange(x.shape[1], device=DEV)[None]
    k = s["top_k"][:, None]
    first = torch.where(t > 0, torch.where((k > 0) & (k < x.shape[1]), k, x.shape[1]), 1)
    among = torch.where(rank < first, sorted_mass, 0)
    before = torch.cumsum(among, 1) - among
    p = s["top_p"][:, None].double()
    keep = (rank < first) & ((before.double() < p * among.sum(1, keepdim=True).double()) | (p >= 1) | (rank == 0)) & (e.gather(1, order) >= s["min_p"][:, None]) & (sorted_mass > 0)
    kept = torch.zeros_like(mass).scatter(1, order, torch.where(keep, sorted_mass, 0))
    total = kept.sum(1)
    want = (s["uniform"].double() * total.double()).long().minimum(total - 1)
    token = torch.searchsorted(torch.cumsum(kept, 1), want[:, None], right=True)
    share = kept.gather(1, token)[:, 0].double() / total.double()
    return dict(token=token[:, 0].int(), probability=share.float(), kept=keep.sum(1, dtype=torch.int32))


def _seen_pairs(case):
    """(query, key) pairs that the masks leave, and keys that at least one query of their request sees."""
    pairs = keys = 0
    for cached, fresh in zip(*_lengths(case)):
        w = case["window"] or cached + fresh
        first = max(0, cached - w + 1)
        keys += cached + fresh - first if fresh else 0
        short = min(fresh, max(0, w - cached))  # the queries whose window reaches the first key
        pairs += short * cached + short * (short + 1) // 2 + (fresh - short) * w
    return pairs, keys


def work(case):
    op = case["op"]
    if op == "plan":
        cached, fresh = _lengths(case)
        n, tokens, page = case["requests"], sum(fresh), case["page"]
        fresh_pages = sum(_pages(c + f, page) - _pages(c, page) for c, f in zip(cached, fresh))
        return dict(bytes=4 * (2 * n + 2 * n + 1 + 3 * (tokens + 5) + 2 * fresh_pages + 3), flops=0)
    if op == "rope":
        t, hq, hk, d = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
        return dict(bytes=t * (8 * hq * d + 12 * hk * d + 4 * case["rotary"] + 8), flops=t * (hq + hk) * (3 * case["rotary"] + (4 * d if case["norm"] else 0)))
    if op == "attend":
        pairs, keys = _seen_pairs(case)
        tokens = sum(_lengths(case)[1])
        return dict(bytes=8 * tokens * case["q_heads"] * case["head_dim"] + 4 * keys * case["kv_heads"] * case["head_dim"] + 4 * _pages(keys, case["page"]), flops=4 * pairs * case["q_heads"] * case["head_dim"])
    return dict(bytes=4 * case["rows"] * (case["vocab"] + 8), flops=4 * case["rows"] * case["vocab"])


# ---- the same in 64 bits -------------------------------------------------------------------------------


def exact(case, seed):
    op = case["op"]
    if op == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    if op == "rope":
        d, hq, hk, half = case["head_dim"], case["q_heads"], case["kv_heads"], case["rotary"] // 2
        angle = s["rotation"].double()[s["positions"].long()]
        turn = torch.complex(angle[:, :half], angle[:, half:])
        a = torch.arange(half, device=DEV) * (1 if case["style"] == "halves" else 2)
        b = a + (half if case["style"] == "halves" else 1)
        heads = []
        for x, gain, n in ((s["q"], s["q_gain"], hq), (s["k"], s["k_gain"], hk)):
            x = x.double().reshape(-1, n, d).clone()
            if gain is not None:
                x *= torch.rsqrt(x.square().sum(-1, keepdim=True) / d + 1e-6) * gain.double()
            z = torch.complex(x[..., a], x[..., b]) * turn[:, None]
            x[..., a], x[..., b] = z.real, z.imag
            heads.append(x)
        k_cache, v_cache = torch.zeros_like(s["k_cache"], dtype=torch.float64), torch.zeros_like(s["v_cache"], dtype=torch.float64)
        block, line = s["slots"].long() // case["page"], s["slots"].long() % case["page"]
        for h in range(hk):
            k_cache[block, h, line], v_cache[block, h, line] = heads[1][:, h], s["v"].double().reshape(-1, hk, d)[:, h]
        return dict(q_out=heads[0].reshape(-1, hq * d), k_cache=k_cache, v_cache=v_cache)
    if op == "attend":
        y = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        group = case["q_heads"] // case["kv_heads"]
        at = 0
        for r, (cached, fresh) in enumerate(zip(*_lengths(case))):
            n = cached + fresh
            used = s["table"][r, : _pages(n, case["page"])].long()
            position = torch.arange(cached, n, device=DEV)[:, None]
            key = torch.arange(n, device=DEV)[None]
            hidden = (key > position) | ((key <= position - case["window"]) if case["window"] else False)
            for h in range(case["kv_heads"]):
                k, v = (c[used, h].reshape(-1, case["head_dim"])[:n].double() for c in (s["k_cache"], s["v_cache"]))
                for g in range(h * group, (h + 1) * group):
                    score = (s["q"][at : at + fresh, g].double() @ k.T * case["head_dim"] ** -0.5).masked_fill(hidden, -math.inf)
                    y[at : at + fresh, g] = torch.softmax(score, 1) @ v
            at += fresh
        return y
    probability = []
    for r in range(case["rows"]):  # weights as they are, not in steps of 2^-40
        x = s["logits"][r].double()
        t = float(s["temperature"][r])
        if t <= 0:
            probability.append(1.0)
            continue
        order = torch.argsort(x, descending=True, stable=True)
        w = torch.exp((x[order] - x.max()) / t)
        if 0 < case["top_k"] < x.numel():
            w[case["top_k"] :] = 0
        p = float(s["top_p"][r])
        if p < 1:
            w = torch.where(torch.cumsum(w, 0) - w < p * w.sum(), w, 0.0)
        w = torch.where(w >= float(s["min_p"][r]), w, 0.0)
        back = torch.zeros_like(x).scatter(0, order, w)
        token = int(torch.searchsorted(torch.cumsum(back, 0), float(s["uniform"][r]) * back.sum(), right=True))
        probability.append(float(back[min(token, x.numel() - 1)] / back.sum()))
    return dict(token=None, probability=torch.tensor(probability, dtype=torch.float64), kept=None)
