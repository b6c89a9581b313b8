"""The operators of a serving step in 64 bits, token by token: what their GPU tests compare with."""
import math

import torch


def pages(n, page):
    return -(-n // page)


def plan(cached, fresh, table, free, page, max_tokens):
    """The same integers with Python loops: (table, starts, lengths, slots, positions, owners, status)."""
    cached, fresh = [max(c, 0) for c in cached], [max(f, 0) for f in fresh]
    table = [list(row) for row in table]
    width, taken, lacking = len(table[0]), 0, 0
    starts, slots, positions, owners = [0], [], [], []
    for r, (c, f) in enumerate(zip(cached, fresh)):
        for column in range(pages(c, page), pages(c + f, page)):
            if column >= width:
                lacking += 1
            elif taken < len(free):
                table[r][column] = free[taken]
                taken += 1
            else:
                table[r][column] = -1
                lacking += 1
        for position in range(c, c + f):
            entry = table[r][position // page] if position // page < width else -1
            slots.append(entry * page + position % page if entry >= 0 else -1)
            positions.append(position)
            owners.append(r)
        starts.append(starts[-1] + f)
    pad = max(0, max_tokens - len(slots))
    status = [starts[-1], taken, lacking]
    return table, starts, [c + f for c, f in zip(cached, fresh)], (slots + [-1] * pad)[:max_tokens], (positions + [0] * pad)[:max_tokens], (owners + [-1] * pad)[:max_tokens], status


def turned(x, gain, epsilon, angles, style):
    """x [tokens, heads, d] in 64 bits: normed and rotated, with the size of each element's pair (what its rounding is relative to)."""
    if gain is not None:
        x = x / (x.square().mean(-1, keepdim=True) + epsilon).sqrt() * gain.double()
    y, size = x.clone(), x.abs().clone()
    half = angles.shape[1] // 2
    cos, sin = angles[:, None, :half].double(), angles[:, None, half:].double()
    at = torch.arange(half, device=x.device)
    a, b = (at, at + half) if style == "halves" else (2 * at, 2 * at + 1)
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, size


def attention(q, k_cache, v_cache, table, starts, lengths, scale, window=0):
    """q [tokens, heads, d]; caches [pages, kv heads, page, d]. Returns y, and for each output the bound that its rounding stays
    under: (4 e + 2^-18) sum w |v| / sum w with e = 2 d 2^-24 max_j scale sum |q k_j|, the most a score in 32 bits is off by."""
    tokens, hq, d = q.shape
    n_pages, hk, page, _ = k_cache.shape
    y, bound = torch.zeros((tokens, hq, d), dtype=torch.float64, device=q.device), torch.zeros((tokens, hq, d), dtype=torch.float64, device=q.device)
    for r in range(len(lengths)):
        for t in range(starts[r], starts[r + 1]):
            position = lengths[r] - (starts[r + 1] - t)
            keys = [j for j in range(max(0, position - window + 1) if window else 0, min(position + 1, lengths[r], table.shape[1] * page))]
            keys = [j for j in keys if 0 <= int(table[r, j // page]) < n_pages]
            if not keys:
                continue
            block = torch.tensor([int(table[r, j // page]) for j in keys], device=q.device)
            line = torch.tensor([j % page for j in keys], device=q.device)
            for h in range(hk):
                mine = slice(h * (hq // hk), (h + 1) * (hq // hk))
                k, v = k_cache[block, h, line].double(), v_cache[block, h, line].double()
                query = q[t, mine].double()
                w = torch.softmax(scale * query @ k.T, 1)
                y[t, mine] = w @ v
                off = 2 * d * 2.0**-24 * scale * (query.abs() @ k.abs().T).amax(1, keepdim=True)
                bound[t, mine] = (4 * off + 2.0**-18) * (w @ v.abs())
    return y, bound


def kept_weights(logits, temperature, top_k, top_p, min_p):
    """A row's weights in 64 bits, zero where a token is not kept, and its tokens by rank."""
    x = [(-math.inf if math.isnan(v) else v) for v in logits]
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    top = x[order[0]]
    if top == -math.inf:
        return [0.0] * len(x), order
    w = [1.0 if v == top else (math.exp((v - top) / temperature) if temperature > 0 and top < math.inf else 0.0) for v in x]
    w = [v if v >= 2.0**-40 else 0.0 for v in w]
    keep = order[: (1 if temperature <= 0 else (top_k if top_k > 0 else len(x)))]
    mass, before, kept = sum(w[i] for i in keep), 0.0, [0.0] * len(x)
    for rank, i in enumerate(keep):
        if (rank == 0 or top_p >= 1 or before < top_p * mass) and w[i] >= min_p:
            kept[i] = w[i]
        before += w[i]
    return kept, order
