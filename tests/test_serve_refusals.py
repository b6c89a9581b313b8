"""What the small decoder of serve.py cannot answer rightly, it refuses before anything is computed (no GPU: the model is a stand-in that has no device)."""
from types import SimpleNamespace

import pytest

from recipe_dev_b200 import serve


@pytest.fixture
def model(monkeypatch):
    torch = pytest.importorskip("torch")
    cpu = torch.device("cpu")
    cache = SimpleNamespace(pages=64)
    random = torch.Generator
    monkeypatch.setattr(torch, "Generator", lambda device=None: random())
    return SimpleNamespace(positions=32, vocabulary=100, page_size=16, device=cpu, layers=[dict(cache=cache)])


@pytest.mark.parametrize("prompts,new,chunk,why", [([], 4, 8, "prompt"), ([[1], []], 4, 8, "prompt"), ([[1, 2]], 0, 8, "new token"), ([[1, 2]], -1, 8, "new token"), ([[1, 2]], 4, 0, "chunks"),
                                                   ([[1] * 30, [1]], 4, 8, "32 positions"), ([[1] * 33], 1, 8, "32 positions"), ([[1, 100]], 4, 8, "0 .. 99"), ([[1, -1]], 4, 8, "0 .. 99")])
def test_refusals(model, prompts, new, chunk, why):
    with pytest.raises(ValueError, match=why):
        serve.Batch(model, prompts, new, chunk)


@pytest.mark.parametrize("prompts,new", [([[1] * 32], 1), ([[1] * 29, [99]], 4), ([[0]], 32)])
def test_the_longest_that_there_are(model, prompts, new):
    batch = serve.Batch(model, prompts, new, 8)
    assert batch.fresh() == [min(8, len(p)) for p in prompts] and batch.table.shape == (len(prompts), max(-(-(len(p) + new) // 16) for p in prompts))
