"""A cache of one device and a context of another: refused before an address of either is handed on (no GPU: both are stand-ins)."""
import pytest

torch = pytest.importorskip("torch")
import recipe_dev_b200 as rq


@pytest.mark.parametrize("call", ["rope_store", "attention"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.int8])
def test_a_cache_of_another_device(call, dtype):
    class Library:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was called")

    class Plane:  # looks like a tensor of device 1
        def __init__(self, like):
            self.like, self.is_cuda, self.device = like, True, torch.device("cuda", 1)

        def get_device(self):
            return 1

        def __getattr__(self, name):
            return getattr(self.like, name)

    ctx = rq.Context.__new__(rq.Context)
    ctx.lib, ctx.handle, ctx.device = Library(), 0, 0
    codes, scales = (Plane(torch.zeros((2, 2, 16, 64), dtype=dtype)) for _ in range(2)), ()
    if dtype is torch.int8:
        scales = (Plane(torch.zeros((2, 2, 16))) for _ in range(2))
    cache = rq.KvCache(*codes, *scales)
    q, ints = Plane(torch.zeros((1, 2 * 64))), Plane(torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="the cache must lie on the context's device"):
        if call == "rope_store":
            ctx.rope_store(q, q, q, ints, ints, None, cache, q_out=q)
        else:
            ctx.attention(q, cache, Plane(torch.zeros((1, 4), dtype=torch.int32)), ints, Plane(torch.ones(1, dtype=torch.int32)), y=q)
    ctx.handle = 0
