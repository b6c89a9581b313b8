"""Attention over queries and keys of any size: what is small in one and large in the other gives scores as any others. GPU only (-m gpu).

The bounds are those of serving_reference.attention, which are relative to scale * sum |q k|: they do not change when a power of two moves from the queries to
the keys."""
import pytest

from tests import serving_reference as ref
from tests.test_gpu_attention import batch, compare, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fresh", [1, 3, 80])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("factor", [1e-6, 1e-3, 2.0**-5, 2e2, 3e6])
def test_sizes_of_queries_over_f16(rq_ctx, fresh, d, factor):
    b = batch([120, 20], [fresh, fresh], 6, 2, d, 16, "f16", seed=3)
    b["q"].mul_(factor)
    if factor == 1e-6:
        b["cache"].k.copy_((b["cache"].k.float() * 1e4).half())  # (65504 is the largest)
        compare(run(rq_ctx, b, scale=25.0 * d**-0.5), b, scale=25.0 * d**-0.5)
    else:
        b["cache"].k.copy_((b["cache"].k.float() / factor).half())
        compare(run(rq_ctx, b), b)


@pytest.mark.parametrize("fresh", [1, 50])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_a_row_that_differs_from_its_neighbours(rq_ctx, fresh, dtype):
    """Rows of zeros, and rows a million times the size of the others over the same keys (whose scores say only which key is the largest)."""
    b = batch([200], [fresh], 8, 2, 128, 16, dtype, seed=5)
    b["q"][:, :128] = 0.0
    b["q"][:, 128:256] *= 1e-5
    b["q"][0, 256:384] = 0.0
    b["q"][0, 256] = 3.0  # one element alone
    compare(run(rq_ctx, b), b)
    b["q"][:, 512:640] *= 1e6
    got = run(rq_ctx, b)
    want, bound = ref.attention(b["q"].reshape(-1, 8, 128), b["cache"].k, b["cache"].v, b["table"], b["starts"], b["lengths"], 128**-0.5)
    near = (got.double() - want).abs() <= bound
    assert near[:, [0, 1, 2, 3, 5, 6, 7]].all() and (got[:, 4].double() - want[:, 4]).norm() <= 1e-5 * want[:, 4].norm()


@pytest.mark.parametrize("fresh", [1, 40])
@pytest.mark.parametrize("scale", [1e-30, 1e-38, 2.0**-20, 3e38])
def test_scales_at_the_ends(rq_ctx, fresh, scale):
    """A scale so small that all keys weigh the same, and the largest one over queries so small that the scores are as ever."""
    b = batch([100], [fresh], 4, 2, 64, 16, "f16", seed=7)
    if scale > 1:
        b["q"].mul_(2.0**-100).mul_(2.0**-30)  # times 3e38: of order one
    compare(run(rq_ctx, b, scale=scale), b, scale=scale)


@pytest.mark.parametrize("fresh", [1, 40])
def test_queries_that_are_not_finite_touch_their_own_row_only(rq_ctx, fresh):
    import torch

    b = batch([100], [fresh], 4, 2, 64, 16, "f16", seed=9)
    clean = run(rq_ctx, b).clone()
    b["q"][0, 3], b["q"][0, 64 + 5] = float("inf"), float("nan")
    got = run(rq_ctx, b)
    assert not torch.isfinite(got[0, :2]).any()
    assert torch.equal(got[0, 2:], clean[0, 2:]) and torch.equal(got[1:], clean[1:])
