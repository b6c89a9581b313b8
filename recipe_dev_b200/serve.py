"""A small decoder that serves a batch of requests over one paged cache: the library's quantised projections with the serving step's four
operators (plan, norm and rotation and store, attention, the next token) around them, on random weights.

    python -m recipe_dev_b200.serve --requests 16 --prompt 700 --new 128

Every step takes the next token of the requests that are past their prompts and the next chunk of the others, in one batch. A step in which
every request brings one token is recorded once and replayed; the plan runs ahead of it, since the list of free pages moves on. Four layers of the default shape and
the head: 16 requests of up to 828 positions 0.84 ms a replayed step, 32 of up to 964 0.98 ms."""
from __future__ import annotations

import argparse
import random

from . import capi


RECORDED = 64  # the most requests whose single-token steps are recorded (what the work areas are reserved for)


class Decoder:
    """Pre-norm layers (norm, attention, residual, norm, gated feed-forward, residual) of Q4_K projections, a Q6_K embedding that is the head too."""

    def __init__(self, ctx: capi.Context, layers: int, hidden: int, q_heads: int, kv_heads: int, head_dim: int, ffn: int, vocabulary: int, pages: int, page_size: int = 16, positions: int = 16384,
                 seed: int = 0, dtype=None):
        import torch

        self.ctx, self.hidden, self.q_heads, self.kv_heads, self.head_dim, self.ffn, self.vocabulary = ctx, hidden, q_heads, kv_heads, head_dim, ffn, vocabulary
        self.page_size, self.device = page_size, torch.device("cuda", ctx.device)
        made = torch.Generator(device=self.device).manual_seed(seed)

        def weight(kind, rows, cols):
            blocks = ctx.quantize(kind, torch.randn(rows * cols, generator=made, device=self.device) * cols**-0.5)
            return ctx.weight_from_device(kind, blocks, rows, cols)

        def gain(n):
            return 1.0 + 0.1 * torch.randn(n, generator=made, device=self.device)

        q, kv = q_heads * head_dim, kv_heads * head_dim
        self.embedding = weight(capi.Q6_K, vocabulary, hidden)
        self.last_gain = gain(hidden)
        self.layers = [dict(qkv=[weight(capi.Q4_K, n, hidden) for n in (q, kv, kv)], o=weight(capi.Q4_K, hidden, q), gate=weight(capi.Q4_K, ffn, hidden), up=weight(capi.Q4_K, ffn, hidden),
                            down=weight(capi.Q4_K, hidden, ffn), gains=[gain(hidden), gain(hidden), gain(head_dim), gain(head_dim)],
                            cache=capi.KvCache.empty(pages, kv_heads, page_size, head_dim, dtype, ctx.device)) for _ in range(layers)]
        self.positions, self.rotation = positions, ctx.rope_table(positions, head_dim)
        ctx.reserve(max(vocabulary, ffn), max(hidden, ffn, q), RECORDED)
        ctx.attention_reserve()

    def planes(self, tokens: int, rows: int):
        """The activations of a step of that many tokens, and the logits of that many of them."""
        import torch

        q, kv = self.q_heads * self.head_dim, self.kv_heads * self.head_dim
        sizes = dict(x=self.hidden, h=self.hidden, qkv=q + 2 * kv, turned=q, y=q, gated=self.ffn, up=self.ffn, delta=self.hidden)
        made = {name: torch.empty((tokens, n), device=self.device) for name, n in sizes.items()}
        made["parts"] = made["qkv"].split([q, kv, kv], dim=1)
        made.update(last=torch.empty((rows, self.hidden), device=self.device), logits=torch.empty((rows, self.vocabulary), device=self.device))
        return made

    def _product(self, w, x, y, stream):
        return self.ctx.matvec(w, x, y, stream=stream) if x.shape[0] <= 8 else self.ctx.matmul(w, x, y, stream=stream)

    def hidden_states(self, ids, batch, max_fresh: int, at, stream=None):
        """ids: int32 [tokens]; batch: the plan's table, starts, lengths, slots and positions; at: planes. The last layer's outputs [tokens, hidden]."""
        import torch

        ctx, x, h, parts = self.ctx, at["x"], at["h"], at["parts"]
        ctx.gather_rows(self.embedding, ids, x, stream=stream)
        for layer in self.layers:
            before, after, q_gain, k_gain = layer["gains"]
            ctx.rmsnorm(x, before, y=h, stream=stream)
            if x.shape[0] <= 8:
                ctx.matvec_multi(layer["qkv"], h, parts, stream=stream)
            else:
                for w, y in zip(layer["qkv"], parts):
                    ctx.matmul(w, h, y, stream=stream)
            ctx.rope_store(*parts, batch["positions"], batch["slots"], self.rotation, layer["cache"], q_gain, k_gain, q_out=at["turned"], stream=stream)
            ctx.attention(at["turned"], layer["cache"], batch["table"], batch["starts"], batch["lengths"], max_fresh=max_fresh, y=at["y"], stream=stream)
            ctx.add(x, self._product(layer["o"], at["y"], at["delta"], stream), x, stream=stream)
            ctx.rmsnorm(x, after, y=h, stream=stream)
            if x.shape[0] <= 8:
                ctx.matvec_glu(layer["gate"], layer["up"], h, at["gated"], stream=stream)
            else:
                ctx.matmul(layer["gate"], h, at["gated"], stream=stream)
                ctx.matmul(layer["up"], h, at["up"], stream=stream)
                with torch.cuda.stream(None if stream is None else torch.cuda.ExternalStream(stream, self.device)):
                    torch.nn.functional.silu(at["gated"], inplace=True).mul_(at["up"])
            ctx.add(x, self._product(layer["down"], at["gated"], at["delta"], stream), x, stream=stream)
        return x

    def logits(self, x, at, stream=None):
        self.ctx.rmsnorm(x, self.last_gain, y=at["last"], stream=stream)
        return self._product(self.embedding, at["last"], at["logits"], stream)


class Batch:
    """Requests that are served together: their lengths, pages and tokens. The model's cache is theirs: one batch at a time."""

    def __init__(self, model: Decoder, prompts, new: int, chunk: int = 512, temperature: float = 0.0, top_k: int = 0, top_p: float = 1.0, seed: int = 0, record: bool = True):
        import torch

        if not prompts or not all(prompts) or new < 1 or chunk < 1:
            raise ValueError("Batch: every request needs a prompt, a new token and chunks of at least one")
        if max(len(p) for p in prompts) + new - 1 > model.positions:  # (the last token is not fed back)
            raise ValueError(f"Batch: the longest request passes the model's {model.positions} positions")
        if not all(0 <= t < model.vocabulary for p in prompts for t in p):
            raise ValueError(f"Batch: a prompt's tokens are 0 .. {model.vocabulary - 1}")
        self.model, self.prompts, self.new, self.chunk, self.record = model, prompts, new, chunk, record
        n, ints = len(prompts), dict(dtype=torch.int32, device=model.device)
        pages = model.layers[0]["cache"].pages
        width = max((len(p) + new + model.page_size - 1) // model.page_size for p in prompts)
        self.cached, self.taken, self.sequence, self.planes = [0] * n, 0, None, None
        self.free = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(**ints)
        self.table = torch.full((n, width), -1, **ints)
        size = n * chunk
        self.batch = dict(table=self.table, starts=torch.empty(n + 1, **ints), lengths=torch.empty(n, **ints), slots=torch.empty(size, **ints), positions=torch.empty(size, **ints))
        self.owners, self.status, self.token, self.counts = torch.empty(size, **ints), torch.empty(3, **ints), torch.zeros(n, **ints), torch.empty((2, n), **ints)
        self.uniform = torch.empty(n, device=model.device)
        self.random = torch.Generator(device=model.device).manual_seed(seed)
        self.filters = dict(temperature=torch.full((n,), temperature, device=model.device), top_k=torch.full((n,), top_k, **ints), top_p=torch.full((n,), top_p, device=model.device))

    def fresh(self):
        """How many tokens each request brings next: a chunk of its prompt, the token sampled last, or none."""
        most = [len(p) + self.new - 1 for p in self.prompts]
        return [min(self.chunk, len(p) - c) if c < len(p) else int(c < m) for p, c, m in zip(self.prompts, self.cached, most)]

    def _one_token_each(self, stream=None):
        x = self.model.hidden_states(self.token, self.batch, 1, self.planes, stream)
        self.last_logits = self.model.logits(x, self.planes, stream)
        self.model.ctx.sample(self.last_logits, self.uniform, **self.filters, token=self.token, stream=stream)

    def step(self):
        """One step; returns which requests' self.token is a new token of theirs, or None when all are done."""
        import torch

        model, ctx, fresh = self.model, self.model.ctx, self.fresh()
        if not any(fresh):
            return None
        self.counts.copy_(torch.tensor([self.cached, fresh], dtype=torch.int32))
        ctx.batch_plan(self.counts[0], self.counts[1], self.table, self.free[self.taken :], model.page_size, owners=self.owners, status=self.status,
                       **{k: v for k, v in self.batch.items() if k != "table"})
        # the pages that the plan took, in its order: the next step's list begins behind them
        self.taken += sum(-(-(c + f) // model.page_size) + -c // model.page_size for c, f in zip(self.cached, fresh))
        if self.taken > self.free.shape[0]:
            raise RuntimeError("the cache has too few pages for these requests")
        torch.rand(self.uniform.shape, generator=self.random, out=self.uniform)
        if all(f == 1 for f in fresh) and all(c >= len(p) for c, p in zip(self.cached, self.prompts)):
            if self.planes is None:
                self.planes = model.planes(len(fresh), len(fresh))
            if self.sequence is not None:
                self.sequence.run()
            else:
                self._one_token_each()  # (what is loaded at first use is loaded before a recording)
                if self.record and len(fresh) <= RECORDED:
                    torch.cuda.synchronize(model.device)
                    self._one_token_each(ctx.sequence_begin())
                    self.sequence = ctx.sequence_end()
        else:
            starts = [sum(fresh[:r]) for r in range(len(fresh) + 1)]
            ids = torch.zeros(starts[-1], dtype=torch.int32)
            sampled = [r for r, p in enumerate(self.prompts) if fresh[r] and self.cached[r] >= len(p)]
            for r, p in enumerate(self.prompts):
                if self.cached[r] < len(p):
                    ids[starts[r] : starts[r + 1]] = torch.tensor(p[self.cached[r] : self.cached[r] + fresh[r]], dtype=torch.int32)
            ids = ids.to(model.device)
            ids[torch.tensor([starts[r] for r in sampled], dtype=torch.long, device=model.device)] = self.token[torch.tensor(sampled, dtype=torch.long, device=model.device)]
            planes = model.planes(starts[-1], len(fresh))
            x = model.hidden_states(ids, self.batch, max(fresh), planes)
            last = torch.tensor([max(s - 1, 0) for s in starts[1:]], device=model.device)
            self.last_logits = model.logits(x[last], planes)
            token = ctx.sample(self.last_logits, self.uniform, **self.filters)
            self.token.copy_(torch.where(self.counts[1] > 0, token, self.token))
        self.cached = [c + f for c, f in zip(self.cached, fresh)]
        return [f > 0 and c >= len(p) for f, c, p in zip(fresh, self.cached, self.prompts)]

    def run(self):
        """All steps: a list of new tokens for each request."""
        steps = []
        while (fresh := self.step()) is not None:
            steps.append((fresh, self.token.clone()))
        out = [[] for _ in self.prompts]
        for fresh, token in steps:
            for r, t in enumerate(token.tolist()):
                if fresh[r]:
                    out[r].append(t)
        self.model.ctx.check()
        return out

    def free_sequence(self) -> None:
        if self.sequence is not None:
            self.sequence.free()
        self.sequence = None


def main() -> None:
    import torch

    ask = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, default, text in (("requests", 16, "requests served together"), ("prompt", 700, "the longest prompt's tokens"), ("new", 128, "new tokens of a request"), ("layers", 4, "layers"),
                                ("hidden", 4096, "width"), ("heads", 32, "query heads"), ("kv-heads", 8, "key and value heads"), ("head-dim", 128, "elements of a head"),
                                ("ffn", 14336, "feed-forward width"), ("vocabulary", 32000, "tokens that there are"), ("chunk", 512, "prompt tokens of a request a step"), ("top-k", 40, "0: all"),
                                ("seed", 0, "of weights, prompts and choices")):
        ask.add_argument("--" + name, type=int, default=default, help=f"{text} ({default})")
    ask.add_argument("--temperature", type=float, default=0.8, help="0: always the likeliest (0.8)")
    ask.add_argument("--top-p", type=float, default=0.95, help="(0.95)")
    a = ask.parse_args()
    rng = random.Random(a.seed)
    prompts = [[rng.randrange(a.vocabulary) for _ in range(rng.randint(max(1, a.prompt // 2), max(1, a.prompt)))] for _ in range(a.requests)]
    ctx = capi.Context(0)
    longest = max(len(p) for p in prompts) + a.new
    model = Decoder(ctx, a.layers, a.hidden, a.heads, a.kv_heads, a.head_dim, a.ffn, a.vocabulary, pages=a.requests * (longest + 15) // 16 + a.requests, positions=longest, seed=a.seed)
    batch = Batch(model, prompts, a.new, a.chunk, a.temperature, a.top_k, a.top_p, a.seed)
    marks = []
    while True:
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        fresh = sum(batch.fresh())
        if batch.step() is None:
            break
        end.record()
        marks.append((fresh, begin, end))
    torch.cuda.synchronize()
    ctx.check()
    replayed = [b.elapsed_time(e) for n, b, e in marks if n == a.requests][2:]
    prompt = sum(n for n, _, _ in marks if n > a.requests)
    if prompt:
        print(f"{prompt} tokens in steps with prompts: {sum(b.elapsed_time(e) for n, b, e in marks if n > a.requests):.2f} ms")
    if replayed:
        print(f"{len(replayed)} replayed steps of {a.requests} tokens: {sum(replayed) / len(replayed):.3f} ms a step, {1e3 * a.requests * len(replayed) / sum(replayed):.0f} tokens/s")
    print("last tokens:", batch.token.tolist())
    batch.free_sequence()
    ctx.close()


if __name__ == "__main__":
    main()
