"""The small decoder's last norm is made once a step, whichever launch makes it (no GPU: the context writes down what it is called for)."""
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")
from recipe_dev_b200 import serve


class Calls:
    """Stands for a context: notes every norm's gain, and marks the plane that it writes."""

    def __init__(self):
        self.gains, self.normed, self.products = [], {}, []

    def rmsnorm(self, x, gain, y=None, stream=None):
        self.gains.append(gain)
        self.normed[y.data_ptr()] = gain
        return y

    def residual_norm(self, x, delta, gain=None, delta_gain=None, residual_scale=1.0, y=None, stream=None):
        return self.rmsnorm(x, gain, y)

    def matvec(self, w, x, y, stream=None):
        self.products.append((w, self.normed.get(x.data_ptr())))
        return y

    def __getattr__(self, name):  # products, the store, attention, the sum: what they compute does not matter here
        return lambda *args, **how: None


@pytest.mark.parametrize("norms", ["before", "both"])
@pytest.mark.parametrize("layers", [0, 1, 3])
def test_each_norm_is_made_once(norms, layers):
    ctx, model = Calls(), serve.Decoder.__new__(serve.Decoder)
    for name, value in dict(ctx=ctx, norms=norms, residual_scale=1.0, hidden=8, q_heads=1, kv_heads=1, head_dim=4, ffn=8, vocabulary=5, device="cpu", embedding="head", last_gain="last", rotation=None).items():
        setattr(model, name, value)
    model.layers = [dict(qkv=[], o="o", gate="gate", up="up", down="down", gains=[f"before {n}", f"after {n}", None, None], cache=None, behind=["a", "b"]) for n in range(layers)]
    at = model.planes(3, 3)
    batch = dict.fromkeys(("positions", "slots", "table", "starts", "lengths"))
    model.logits(model.hidden_states(torch.zeros(3, dtype=torch.int32), batch, 1, at), at)
    assert ctx.gains == [f"{side} {n}" for n in range(layers) for side in ("before", "after")] + ["last"]
    assert ctx.products[-1] == ("head", "last")
