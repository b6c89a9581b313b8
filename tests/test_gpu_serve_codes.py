"""The small decoder of serve.py over an 8-bit cache, with norms on both sides of the blocks and log probabilities of its tokens, against the same layers in 64 bits. GPU only (-m gpu)."""
import random

import pytest

pytestmark = pytest.mark.gpu
PROMPTS = [1, 37, 90, 16, 3]


@pytest.fixture(scope="module")
def model():
    import torch

    import recipe_dev_b200 as rq
    from recipe_dev_b200 import serve

    ctx = rq.Context(0)
    yield serve.Decoder(ctx, layers=2, hidden=512, q_heads=8, kv_heads=2, head_dim=64, ffn=768, vocabulary=1000, pages=60, page_size=16, positions=256, dtype=torch.int8, norms="both", residual_scale=0.5)
    ctx.close()


def reference(model, tokens):
    """The logits after the last of these tokens: one sequence, contiguous, 64 bits; keys and values as codes of their heads' steps."""
    import torch

    ctx, d, hq, hk = model.ctx, model.head_dim, model.q_heads, model.kv_heads

    def wide(w):
        return ctx.dequant(w).double()

    def norm(x, gain):
        return x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * gain.double()

    def held(x):
        step = x.abs().amax(-1, keepdim=True) / 127
        return (x / step).round() * step

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
        k, v = (held(a).repeat_interleave(hq // hk, 1) for a in (k, v.view(n, hk, d)))
        scores = torch.einsum("ihd,jhd->hij", q, k) * d**-0.5
        scores.masked_fill_(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), float("-inf"))
        x = x + 0.5 * norm(torch.einsum("hij,jhd->ihd", scores.softmax(-1), v).reshape(n, -1) @ wide(layer["o"]).T, layer["behind"][0])
        h = norm(x, after)
        x = x + 0.5 * norm((torch.nn.functional.silu(h @ wide(layer["gate"]).T) * (h @ wide(layer["up"]).T)) @ wide(layer["down"]).T, layer["behind"][1])
    return norm(x[-1:], model.last_gain)[0] @ embedding.T


def test_every_step_against_64_bits(model):
    """Every logit of every step, and the log probabilities that come with the tokens.

    The products are good for 1e-3 of a row's size, and there are six in a layer, one after another, and the head: 13 * 1e-3 of the logits' norm. A key or value that lies within its own
    1e-3 of a border between two codes may have the other one, a step, 1 / 127 of its head's largest: a 64th of the elements at most, 1e-3 of a head's size in the
    2-norm, for keys and for values of two layers: 4e-3 more. A log probability is off by no more than twice the largest logit's error."""
    import torch

    from recipe_dev_b200 import serve

    rng = random.Random(1)
    served = serve.Batch(model, [[rng.randrange(model.vocabulary) for _ in range(n)] for n in PROMPTS], new=9, chunk=24, logprobs=3)
    seen = [list(p) for p in served.prompts]
    steps = 0
    while (fresh := served.step()) is not None:
        steps += 1
        for r in range(len(seen)):
            if fresh[r]:
                want, got = reference(model, seen[r]), served.last_logits[r].double()
                assert (got - want).norm() <= 17e-3 * want.norm(), (steps, r)
                seen[r].append(int(served.token[r]))
                assert seen[r][-1] == int(served.last_logits[r].argmax())  # temperature 0
                logp = torch.log_softmax(got, 0)
                assert abs(float(served.scored["logprob"][r]) - float(logp[seen[r][-1]])) <= 1e-5
                assert served.scored["top_token"][r].tolist() == torch.topk(logp, 3).indices.tolist() and served.scored["top_token"][r, 0] == seen[r][-1]
                assert (served.scored["top_logprob"][r].double() - torch.topk(logp, 3).values).abs().max() <= 1e-5
    assert [len(s) - n for s, n in zip(seen, PROMPTS)] == [9] * len(PROMPTS)
    served.free_sequence()
    model.ctx.check()


@pytest.mark.parametrize("requests", [3, 11])
def test_replayed_steps_give_the_direct_steps_tokens_and_scores(model, requests):
    from recipe_dev_b200 import serve

    def run(record):
        served = serve.Batch(model, [[5 + r, 6, 7] for r in range(requests)], new=20, record=record, temperature=0.9, top_k=50, top_p=0.9, seed=3, logprobs=2)
        out = served.run()
        assert (served.sequence is not None) == record
        served.free_sequence()
        return out, served.scores

    direct, scores = run(False)
    assert run(True) == (direct, scores) and all(len(t) == 20 for t in direct)
    for tokens, of in zip(direct, scores):
        assert len(of) == 20
        for token, (logprob, likeliest) in zip(tokens, of):
            assert likeliest[0][1] >= likeliest[1][1] >= -30 and logprob <= likeliest[0][1] <= 0
            assert all(logprob == other for t, other in likeliest if t == token)


def test_scores_are_none_unless_asked_for(model):
    from recipe_dev_b200 import serve

    served = serve.Batch(model, [[1, 2]], new=3)
    assert len(served.run()[0]) == 3 and served.scores is None
    served.free_sequence()
    served = serve.Batch(model, [[1, 2]], new=3, logprobs=0)
    served.run()
    assert [likeliest for _, likeliest in served.scores[0]] == [[], [], []]
    served.free_sequence()
