"""The small decoder of serve.py, all of the serving step's operators together, against the same layers in 64 bits. GPU only (-m gpu)."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    import recipe_dev_b200 as rq
    from recipe_dev_b200 import serve

    ctx = rq.Context(0)
    yield serve.Decoder(ctx, layers=2, hidden=512, q_heads=8, kv_heads=2, head_dim=64, ffn=768, vocabulary=1000, pages=60, page_size=16, positions=256)
    ctx.close()


def reference(model, tokens):
    """The logits after the last of these tokens: one sequence, contiguous, 64 bits; keys and values rounded to the cache's type."""
    import torch

    ctx, d, hq, hk = model.ctx, model.head_dim, model.q_heads, model.kv_heads

    def wide(w):
        return ctx.dequant(w).double()

    def norm(x, gain):
        return x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * gain.double()

    n = len(tokens)
    angle = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    c, s = angle.cos()[:, None], angle.sin()[:, None]

    def turn(x):
        a, b = x[..., : d // 2], x[..., d // 2 :]
        return torch.cat([a * c - b * s, a * s + b * c], -1)

    embedding = wide(model.embedding)
    x = embedding[torch.tensor(tokens, device="cuda")]
    for layer in model.layers:
        before, after, q_gain, k_gain = layer["gains"]
        q, k, v = (norm(x, before) @ wide(w).T for w in layer["qkv"])
        q, k = turn(norm(q.view(n, hq, d), q_gain)), turn(norm(k.view(n, hk, d), k_gain))
        k, v = (a.float().to(layer["cache"].k.dtype).double().repeat_interleave(hq // hk, 1) for a in (k, v.view(n, hk, d)))
        scores = torch.einsum("ihd,jhd->hij", q, k) * d**-0.5
        scores.masked_fill_(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), float("-inf"))
        x = x + torch.einsum("hij,jhd->ihd", scores.softmax(-1), v).reshape(n, -1) @ wide(layer["o"]).T
        h = norm(x, after)
        x = x + (torch.nn.functional.silu(h @ wide(layer["gate"]).T) * (h @ wide(layer["up"]).T)) @ wide(layer["down"]).T
    return norm(x[-1:], model.last_gain)[0] @ embedding.T


PROMPTS = [1, 37, 90, 16, 3]


def batch(model, **how):
    import random

    from recipe_dev_b200 import serve

    rng = random.Random(1)
    return serve.Batch(model, [[rng.randrange(model.vocabulary) for _ in range(n)] for n in PROMPTS], new=9, chunk=24, **how)


def test_every_step_against_64_bits(model):
    """Every logit of every step of a batch whose requests pass from chunks of prompts to single tokens at different times.

    The products are good for 1e-3 of a row's size where the framework promises least (its parity tests' bound), and there are six in a
    layer, one after another, and the head: 13 * 1e-3 of the logits' norm, which what is stored in 16 bits (a rounding to the other side, 2^-10 of
    single elements) is below."""
    served = batch(model)
    seen = [list(p) for p in served.prompts]
    steps = 0
    while (fresh := served.step()) is not None:
        steps += 1
        for r in range(len(seen)):
            if fresh[r]:
                want = reference(model, seen[r])
                got = served.last_logits[r].double()
                assert (got - want).norm() <= 13e-3 * want.norm(), (steps, r)
                seen[r].append(int(served.token[r]))
                assert seen[r][-1] == int(served.last_logits[r].argmax())  # temperature 0
    assert [len(s) - n for s, n in zip(seen, PROMPTS)] == [9] * len(PROMPTS)
    served.free_sequence()
    model.ctx.check()


@pytest.mark.parametrize("requests", [3, 11])
@pytest.mark.parametrize("filters", [dict(), dict(temperature=0.9, top_k=50, top_p=0.9, seed=3)])
def test_replayed_steps_give_the_direct_steps_tokens(model, filters, requests):
    def run(record):
        from recipe_dev_b200 import serve

        served = serve.Batch(model, [[5 + r, 6, 7] for r in range(requests)], new=20, record=record, **filters)
        out = served.run()
        assert (served.sequence is not None) == record
        served.free_sequence()
        return out

    direct = run(False)
    assert run(True) == direct and all(len(t) == 20 for t in direct)


def test_too_few_pages(model):
    from recipe_dev_b200 import serve

    served = serve.Batch(model, [[1] * 200] * 5, new=2, chunk=512)
    with pytest.raises(RuntimeError, match="too few pages"):
        served.run()
    model.ctx.check()
