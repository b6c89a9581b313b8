"""More operators of a serving step, as cases that can be timed: the store of rotated keys and of values into a cache of 8-bit codes with
a scale for each token and head, attention over that cache, the log probabilities of given tokens with entropy and likeliest alternatives,
and the step from one block to the next (norm behind a block, gate, residual sum, norm in front of the next block).

Where `own` is false, `run` computes them with elementary torch operations in 32 bits (64 for what is rounded to a code); where it is
true, through recipe_dev_b200.Context as a host program calls it. Inputs are made on the GPU from the seed alone; lengths follow from the
case, so that a case always is the same amount of work. `exact` gives the same results in 64 bits from the definitions.
"""
import math

import torch

own = False

DEV = "cuda:0"
_contexts = {}


def listed():
    llama = dict(q_heads=32, kv_heads=8, head_dim=128)
    return [
        # One decoded token's queries, keys and values: the smallest call.
        dict(name="store_one", op="store", tokens=1, style="pairs", norm=False, rotary=128, page=16, **llama),
        # A prompt of ragged length, with a norm for each head.
        dict(name="store_prompt", op="store", tokens=2039, style="halves", norm=True, rotary=128, page=16, **llama),
        # One decoded token over a short conversation: latency.
        dict(name="attend_one", op="attend", requests=1, cached_lo=1000, cached_hi=1000, fresh_lo=1, fresh_hi=1, page=16, window=0, **llama),
        # One decoded token at the end of a long document: the cache is read once, by the whole GPU.
        dict(name="attend_long", op="attend", requests=1, cached_lo=131070, cached_hi=131070, fresh_lo=1, fresh_hi=1, page=64, window=0, **llama),
        # 64 sequences of uneven length decoded together.
        dict(name="attend_batch", op="attend", requests=64, cached_lo=0, cached_hi=8191, fresh_lo=1, fresh_hi=1, page=16, window=0, **llama),
        # A chunk of a long prompt: 509 new tokens over what earlier chunks left in the cache.
        dict(name="attend_chunk", op="attend", requests=1, cached_lo=7680, cached_hi=7680, fresh_lo=509, fresh_hi=509, page=16, window=0, **llama),
        # Whole prompts of uneven length.
        dict(name="attend_prompts", op="attend", requests=4, cached_lo=0, cached_hi=0, fresh_lo=1021, fresh_hi=3001, page=16, window=0, **llama),
        # A decoded batch's tokens with twenty alternatives each, over a large vocabulary.
        dict(name="logprobs_batch", op="logprobs", rows=64, vocab=262144, top=20, spread=2.5),
        # A prompt's tokens scored, without alternatives.
        dict(name="logprobs_prompt", op="logprobs", rows=2039, vocab=32000, top=0, spread=2.5),
        # One decoded token between two blocks: latency.
        dict(name="join_one", op="join", tokens=1, width=4096, behind=False, gate="none"),
        # 64 decoded tokens through blocks with norms on both sides.
        dict(name="join_batch", op="join", tokens=64, width=2560, behind=True, gate="none"),
        # A prompt of ragged length, norms on both sides and a gate for each element.
        dict(name="join_prompt", op="join", tokens=2039, width=4096, behind=True, gate="elements"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "store", "attend", "attend", "attend", "attend", "logprobs", "logprobs", "join", "join"])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    if op == "logprobs":
        vocab = _log(rng, 1000, 262144)
        return dict(op=op, rows=_log(rng, 1, max(1, min(4096, 64_000_000 // vocab))), vocab=vocab, top=rng.choice([0, 0, 1, 5, 20, 20, 64]), spread=rng.uniform(1.0, 5.0))
    if op == "join":
        return dict(op=op, tokens=_log(rng, 1, 2000), width=rng.choice([1024, 2048, 2560, 2816, 4096, 4096, 5000]), behind=rng.random() < 0.6, gate=rng.choice(["none", "none", "channels", "tokens", "elements"]))
    heads = dict(rng.choice([dict(q_heads=32, kv_heads=8, head_dim=128), dict(q_heads=32, kv_heads=8, head_dim=128), dict(q_heads=16, kv_heads=16, head_dim=64), dict(q_heads=28, kv_heads=4, head_dim=128),
                             dict(q_heads=8, kv_heads=4, head_dim=256), dict(q_heads=40, kv_heads=2, head_dim=64)]))
    if op == "store":
        rotary = heads["head_dim"] if rng.random() < 0.75 else heads["head_dim"] // 2
        return dict(op=op, tokens=_log(rng, 1, 4096), style=rng.choice(["halves", "pairs"]), norm=rng.random() < 0.6, rotary=rotary, page=page, **heads)
    width = heads["kv_heads"] * heads["head_dim"]
    case = dict(op=op, page=page, window=rng.choice([0, 0, 0, 128, 1000]), **heads)
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
    op, gen = case["op"], _gen(seed, 0)
    if op == "store":
        t, hq, hk, d, page = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
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
        s["k_cache"], s["v_cache"] = (torch.zeros((pages, hk, page, d), dtype=torch.int8, device=DEV) for _ in range(2))
        s["k_scale"], s["v_scale"] = (torch.zeros((pages, hk, page), device=DEV) for _ in range(2))
        s["k_values"], s["v_values"] = (torch.empty((pages, hk, page, d), dtype=torch.float16, device=DEV) for _ in range(2))
        s["q_out"] = torch.empty((t, hq * d), device=DEV)
    elif op == "attend":
        cached, fresh = _lengths(case)
        hq, hk, d, page, n = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], case["requests"]
        held = [_pages(c + f, page) for c, f in zip(cached, fresh)]
        pages, t = sum(held) + 3, sum(fresh)
        s["table"] = torch.full((n, max(held) + 1), -1, dtype=torch.int32, device=DEV)
        mine = torch.arange(max(held) + 1, device=DEV)[None] < torch.tensor(held, device=DEV)[:, None]
        s["table"][mine] = torch.randperm(pages, generator=gen, device=DEV).int()[: sum(held)]
        # codes of normal keys and values, whose sizes differ from token to token
        s["k_cache"], s["v_cache"] = (torch.empty((pages, hk, page, d), device=DEV).normal_(0.0, 42.0, generator=gen).round_().clamp_(-127, 127).to(torch.int8) for _ in range(2))
        s["k_scale"], s["v_scale"] = (torch.exp(0.3 * torch.randn((pages, hk, page), generator=gen, device=DEV)) / 42.0 for _ in range(2))
        # some heads look around evenly, some at a few tokens
        s["q"] = torch.randn((t, hq, d), generator=gen, device=DEV) * torch.linspace(0.5, 3.0, hq, device=DEV)[:, None]
        s["starts"], s["lengths"] = _int([sum(fresh[:i]) for i in range(n + 1)]), _int([c + f for c, f in zip(cached, fresh)])
        s["max_fresh"], s["longest"], s["scale"] = max(fresh), max(c + f for c, f in zip(cached, fresh)), d**-0.5
        s["y"] = torch.empty((t, hq, d), device=DEV)
    elif op == "logprobs":
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        s["logits"] = case["spread"] * torch.randn((rows, vocab), generator=gen, device=DEV)
        # a text's own tokens are likely ones, mostly: the best of a few
        guesses = torch.randint(0, vocab, (rows, 512), generator=gen, device=DEV)
        s["token"] = guesses.gather(1, s["logits"].gather(1, guesses).argmax(1, keepdim=True))[:, 0].int()
        s["logprob"], s["entropy"] = (torch.empty(rows, device=DEV) for _ in range(2))
        s["rank"] = torch.empty(rows, dtype=torch.int32, device=DEV)
        s["top_token"], s["top_logprob"] = (torch.empty((rows, top), dtype=torch.int32, device=DEV), torch.empty((rows, top), device=DEV)) if top else (None, None)
    else:
        t, n = case["tokens"], case["width"]
        s["x"] = 3.0 * torch.randn((t, n), generator=gen, device=DEV)
        s["delta"] = torch.randn((t, n), generator=gen, device=DEV) * torch.exp(0.3 * torch.randn((1, n), generator=gen, device=DEV))
        s["gain"], s["delta_gain"] = 1.0 + 0.2 * torch.randn((2, n), generator=gen, device=DEV)
        if not case["behind"]:
            s["delta_gain"] = None
        shape = {"none": None, "channels": (n,), "tokens": (t, 1), "elements": (t, n)}[case["gate"]]
        s["gate"] = None if shape is None else torch.sigmoid(torch.randn(shape, generator=gen, device=DEV))
        s["residual"] = 0.22 if case["gate"] == "none" else 1.0
        s["x_out"], s["y"] = (torch.empty((t, n), device=DEV) for _ in range(2))
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
        s["handle"] = rq.KvCache(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    return s["handle"]


def _stored(s):
    """What the store leaves: the scales, and the codes as the values that they stand for (to the eleven bits that more than hold a code's seven)."""
    torch.mul(s["k_cache"], s["k_scale"][..., None], out=s["k_values"])
    torch.mul(s["v_cache"], s["v_scale"][..., None], out=s["v_values"])
    return {k: s[k] for k in ("q_out", "k_values", "v_values", "k_scale", "v_scale")}


def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return {"store": _plain_store, "attend": _plain_attend, "logprobs": _plain_logprobs, "join": _plain_join}[op](s, case)
    ctx = _context()
    if op == "store":
        ctx.rope_store(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["rotation"], _cache(s), q_gain=s["q_gain"], k_gain=s["k_gain"], epsilon=1e-6, style=case["style"], q_out=s["q_out"])
        return _stored(s)
    if op == "attend":
        return ctx.attention(s["q"], _cache(s), s["table"], s["starts"], s["lengths"], scale=s["scale"], window=case["window"], max_fresh=s["max_fresh"], y=s["y"])
    if op == "logprobs":
        out = ("logprob", "entropy", "rank", "top_token", "top_logprob")
        ctx.logprobs(s["logits"], s["token"], **{k: s[k] for k in out})
        return {k: s[k] for k in out if s[k] is not None}
    ctx.residual_norm(s["x"], s["delta"], s["gain"], delta_gain=s["delta_gain"], gate=s["gate"], residual_scale=s["residual"], epsilon=1e-6, x_out=s["x_out"], y=s["y"])
    return {k: s[k] for k in ("x_out", "y")}


def _plain_store(s, case):
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
    for name, x in (("k", turned(s["k"].double(), s["k_gain"])), ("v", s["v"].double().reshape(t, -1, d))):  # in 64 bits: codes lie next to borders
        scale = (x.abs().amax(-1, keepdim=True) / 127.0).float()
        s[name + "_cache"][slots // page, :, slots % page] = torch.round(x / torch.where(scale > 0, scale, 1.0)).to(torch.int8)
        s[name + "_scale"][slots // page, :, slots % page] = scale[..., 0]
    s["q_out"].copy_(turned(s["q"], s["q_gain"]).reshape(t, -1))
    return _stored(s)


def _plain_attend(s, case):
    hq, hk, d, page, n = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], case["requests"]
    group, f, longest = hq // hk, s["max_fresh"], s["longest"]
    starts, lengths = s["starts"].long(), s["lengths"].long()
    key = torch.arange(longest, device=DEV)
    block = torch.gather(s["table"].long(), 1, (key // page)[None].expand(n, -1).clamp(max=s["table"].shape[1] - 1)).clamp(min=0)
    line = (key % page)[None]
    k, v = ((c[block, :, line].float() * z[block, :, line][..., None]).transpose(1, 2) for c, z in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])))  # [requests, heads, keys, d]
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


def _plain_logprobs(s, case):
    x, token, k = s["logits"], s["token"].long()[:, None], case["top"]
    down = x - x.amax(1, keepdim=True)
    e = torch.exp(down)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    mine = x.gather(1, token)
    index = torch.arange(x.shape[1], device=DEV)[None]
    out = dict(logprob=(down.gather(1, token) - log_total)[:, 0], entropy=(log_total - (e * down).sum(1, keepdim=True) / total)[:, 0])
    out["rank"] = ((x > mine) | ((x == mine) & (index < token))).sum(1, dtype=torch.int32)
    if k:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
        out |= dict(top_token=order.int(), top_logprob=down.gather(1, order) - log_total)
    return out


def _plain_join(s, case):
    def normed(x, gain):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gain

    delta = s["delta"] if s["delta_gain"] is None else normed(s["delta"], s["delta_gain"])
    if s["gate"] is not None:
        delta = delta * s["gate"]
    x = s["x"] + s["residual"] * delta
    return dict(x_out=x, y=normed(x, s["gain"]))


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
    if op == "store":
        t, hq, hk, d = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
        return dict(bytes=t * (8 * hq * d + hk * (10 * d + 8) + 4 * case["rotary"] + 8), flops=t * ((hq + hk) * (3 * case["rotary"] + (4 * d if case["norm"] else 0)) + 4 * hk * d))
    if op == "attend":
        pairs, keys = _seen_pairs(case)
        tokens = sum(_lengths(case)[1])
        return dict(bytes=8 * tokens * case["q_heads"] * case["head_dim"] + 2 * keys * case["kv_heads"] * (case["head_dim"] + 4) + 4 * _pages(keys, case["page"]), flops=4 * pairs * case["q_heads"] * case["head_dim"])
    if op == "logprobs":
        return dict(bytes=case["rows"] * (4 * case["vocab"] + 16 + 8 * case["top"]), flops=6 * case["rows"] * case["vocab"])
    t, n = case["tokens"], case["width"]
    gate = {"none": 0, "channels": n, "tokens": t, "elements": t * n}[case["gate"]]
    return dict(bytes=16 * t * n + 4 * gate + 4 * n * (1 + case["behind"]), flops=t * n * (6 + 4 * case["behind"] + (case["gate"] != "none")))


# ---- the same in 64 bits -------------------------------------------------------------------------------


def exact(case, seed):
    op = case["op"]
    s = prepare(case, seed)
    if op == "store":
        d, hq, hk, half, page = case["head_dim"], case["q_heads"], case["kv_heads"], case["rotary"] // 2, case["page"]
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
        out = dict(q_out=heads[0].reshape(-1, hq * d))
        block, line = s["slots"].long() // page, s["slots"].long() % page
        for name, x in (("k", heads[1]), ("v", s["v"].double().reshape(-1, hk, d))):
            values, scales = torch.zeros(s["k_cache"].shape, dtype=torch.float64, device=DEV), torch.zeros(s["k_scale"].shape, dtype=torch.float64, device=DEV)
            step = x.abs().max(dim=2).values / 127
            code = torch.where(step[..., None] > 0, x / step[..., None], 0.0).round()
            for h in range(hk):
                values[block, h, line], scales[block, h, line] = code[:, h] * step[:, h, None], step[:, h]
            out |= {name + "_values": values, name + "_scale": scales}
        return out
    if op == "attend":
        y = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        group, d = case["q_heads"] // case["kv_heads"], case["head_dim"]
        at = 0
        for r, (cached, fresh) in enumerate(zip(*_lengths(case))):
            n = cached + fresh
            used = s["table"][r, : _pages(n, case["page"])].long()
            position = torch.arange(cached, n, device=DEV)[:, None]
            key = torch.arange(n, device=DEV)[None]
            hidden = (key > position) | ((key <= position - case["window"]) if case["window"] else False)
            for h in range(case["kv_heads"]):
                k, v = ((c[used, h].double() * z[used, h].double().unsqueeze(-1)).reshape(-1, d)[:n] for c, z in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])))
                for g in range(h * group, (h + 1) * group):
                    score = (s["q"][at : at + fresh, g].double() @ k.T * d**-0.5).masked_fill(hidden, -math.inf)
                    y[at : at + fresh, g] = torch.softmax(score, 1) @ v
            at += fresh
        return y
    if op == "logprobs":
        out = dict(logprob=[], entropy=[], rank=None)
        if case["top"]:
            out |= dict(top_token=None, top_logprob=[])
        for x, token in zip(s["logits"], s["token"].long()):
            logp = torch.log_softmax(x.double(), 0)
            out["logprob"].append(logp[token])
            out["entropy"].append(-(logp.exp() * logp).sum())
            if case["top"]:
                out["top_logprob"].append(torch.topk(logp, case["top"]).values)
        return {k: torch.stack(v) if v is not None else None for k, v in out.items()}
    x, delta = s["x"].double(), s["delta"].double()
    if s["delta_gain"] is not None:
        delta = torch.nn.functional.rms_norm(delta, (case["width"],), s["delta_gain"].double(), 1e-6)
    if s["gate"] is not None:
        delta = torch.mul(delta, s["gate"].double())
    x = torch.add(x, delta, alpha=s["residual"])
    return dict(x_out=x, y=torch.nn.functional.rms_norm(x, (case["width"],), s["gain"].double(), 1e-6))
