"""Attention over 8-bit codes: batches that are longer than the call's arrays, many requests, decode steps among prompts, and every form of the tensor-core kernel. GPU only (-m gpu).

Bounds: as in test_gpu_int8_cache.py."""
import pytest

from tests import serving_reference as ref
from tests.test_gpu_int8_cache import batch, compare, run, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fresh", [[1] * 5, [3, 40, 1, 1, 30]])
def test_a_batch_that_is_longer_than_its_arrays(rq_ctx, fresh):
    """Tokens that the call has no queries for are passed over, and what lies behind the last one stays."""
    import torch

    b = batch([20, 3, 64, 100, 7], fresh, 4, 2, 128, 16)
    there = sum(fresh) - 2
    want, bound = ref.attention(b["q"].reshape(-1, 4, 128), values(b["cache"], "k"), values(b["cache"], "v"), b["table"], b["starts"], b["lengths"], 128**-0.5, 0)
    y = torch.full((sum(fresh), 4 * 128), 9.0, device="cuda")
    short = dict(b, q=b["q"][:there])
    run(rq_ctx, short, max_fresh=max(fresh), y=y[:there])
    assert ((y[:there].reshape(-1, 4, 128).double() - want[:there]).abs() <= bound[:there]).all() and (y[there:] == 9.0).all()


@pytest.mark.parametrize("requests", [129, 700])
@pytest.mark.parametrize("fresh", [1, 26])
def test_many_requests(rq_ctx, requests, fresh):
    """More requests than threads add up at a time; 26 tokens of two heads a key head go to the tensor cores."""
    import torch

    cached = [(37 * r) % 50 for r in range(requests)]
    b = batch(cached, [fresh] * requests, 2, 1, 64, 8)
    got = run(rq_ctx, b)
    some = [0, 1, 64, requests // 2, requests - 1]
    for r in some:
        mine = slice(r * fresh, (r + 1) * fresh)
        compare(got[mine].contiguous(), dict(b, q=b["q"][mine], table=b["table"][r : r + 1], starts=[0, fresh], lengths=[cached[r] + fresh]), norm=None)
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (8, 2, 128), (16, 1, 128)])
@pytest.mark.parametrize("fresh", [25, 33, 64])
@pytest.mark.parametrize("page", [8, 16, 128])
@pytest.mark.parametrize("window", [0, 50])
def test_forms_of_the_tensor_core_kernel(rq_ctx, hq, hk, d, fresh, page, window):
    """One tile of rows whose pipes take alternate keys, and two tiles that share keys; pages of half a copy, of one, and of eight."""
    b = batch([0, 170, 128], [fresh, fresh, 5], hq, hk, d, page, seed=page)
    compare(run(rq_ctx, b, window=window), b, window=window)


@pytest.mark.parametrize("fresh", [[1, 300, 1, 0, 2], [200, 1, 1, 1, 1], [1, 1, 1, 1, 64]])
@pytest.mark.parametrize("hq,hk", [(8, 2), (4, 4)])
def test_decode_steps_among_prompts(rq_ctx, fresh, hq, hk):
    b = batch([500, 3, 129, 60, 0], fresh, hq, hk, 128, 16)
    compare(run(rq_ctx, b), b)


def test_uneven_tiles_beside_even_ones(rq_ctx):
    """Scales that differ by more than a row's headroom in some tiles and not in others, masked and not, over several blocks of rows."""
    b = batch([400], [150], 4, 2, 128, 16)
    c = b["cache"]
    for entry in (3, 4, 12, 30):
        c.v_scale[int(b["table"][0, entry]), :, 5] *= 2.0**20
    c.v_scale[int(b["table"][0, 20])] *= 2.0**-25
    compare(run(rq_ctx, b), b, norm=None)


def test_two_recordings_over_one_work_area(rq_ctx):
    """Both a long decode step, whose rows many CTAs have parts of, replayed one after another and in turn."""
    import torch

    b = [batch([6000 + 900 * i], [1], 8, 2, 128, 16, seed=i) for i in range(2)]
    y = [torch.zeros_like(x["q"]) for x in b]
    ints = [[torch.tensor(x[k], dtype=torch.int32, device="cuda") for k in ("starts", "lengths")] for x in b]
    rq_ctx.attention_reserve()
    want = [run(rq_ctx, x).clone() for x in b]
    sequences = []
    for x, out, (starts, lengths) in zip(b, y, ints):
        torch.cuda.synchronize()
        rq_ctx.attention(x["q"], x["cache"], x["table"], starts, lengths, max_fresh=1, y=out, stream=rq_ctx.sequence_begin())
        sequences.append(rq_ctx.sequence_end())
    for turn in (0, 1, 1, 0, 1):
        y[turn].zero_()
        sequences[turn].run()
        torch.cuda.synchronize()
        assert torch.equal(y[turn].reshape(want[turn].shape), want[turn])
    for s in sequences:
        s.free()
    rq_ctx.check()
