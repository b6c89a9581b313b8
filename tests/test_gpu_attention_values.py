"""Attention over values of any size that the cache holds. GPU only (-m gpu)."""
import pytest

from tests.test_gpu_attention import batch, compare, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fresh", [1, 7, 60])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_values_near_the_end_of_bf16(rq_ctx, fresh, d):
    """Values of 1e36 over a few keys: no sum of the formula's passes what fp32 holds."""
    b = batch([5], [fresh], 4, 2, d, 16, "bf16", seed=11)
    b["q"].mul_(0.3)  # flat heads: no sum of weights is above the number of keys
    b["cache"].v.copy_((b["cache"].v.float() * 1e36).bfloat16())
    compare(run(rq_ctx, b), b)
