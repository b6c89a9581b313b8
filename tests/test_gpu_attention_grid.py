"""How many CTAs a call is dealt out to depends on the call alone, so that its bits do not depend on which calls came before. GPU only (-m gpu)."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import sys
import torch
import recipe_dev_b200 as rq

ctx = rq.Context(0)
gen = torch.Generator(device="cuda").manual_seed(1)
i32 = dict(dtype=torch.int32, device="cuda")
made = {}
for kind in (torch.float16, torch.bfloat16):
    for d in (64, 128, 256):
        cache = rq.KvCache(*((torch.randn((512, 2, 64, d), generator=gen, device="cuda").to(kind)) for _ in range(2)))
        table = torch.arange(512, **i32)[None]
        made[d, kind] = (cache, table, torch.randn((4, 4, d), generator=gen, device="cuda"))

def call(d, kind, requests):
    cache, table, q = made[d, kind]
    if requests > 1:
        n = requests
        return ctx.attention(q[:1].expand(n, 4, d).contiguous(), cache, table.expand(n, 512).contiguous(), torch.arange(n + 1, **i32), torch.ones(n, **i32), max_fresh=1)
    return ctx.attention(q, cache, table, torch.tensor([0, 4], **i32), torch.tensor([32768], **i32), max_fresh=4)

for first in map(int, sys.argv[1].split(",")):
    for at in made:
        call(*at, first)
ctx.check()
print([float(call(*at, 1).double().sin().sum()) for at in made], [call(*at, 1).view(torch.int32).long().mul(2654435761).remainder(1000003).sum().item() for at in made])
ctx.check()
"""


def after(first):
    run = subprocess.run([sys.executable, "-c", PROGRAM, first], capture_output=True, text=True, timeout=300, cwd=Path(__file__).resolve().parent.parent, env=dict(os.environ))
    assert run.returncode == 0, run.stderr[-2000:]
    return run.stdout.strip().splitlines()[-1]


def test_a_call_gives_the_same_bits_whatever_came_first():
    want = after("1")
    assert after("4096") == want
    assert after("700,1,64") == want


@pytest.mark.parametrize("fresh", [1, 40])
def test_calls_after_a_reported_wait(fresh):
    """A check that reports a wait that ran out clears the context's counts of parts; rows dealt out over many CTAs are the same before and after."""
    import torch

    import recipe_dev_b200 as rq

    ctx = rq.Context(0)
    gen = torch.Generator(device="cuda").manual_seed(3)
    i32 = dict(dtype=torch.int32, device="cuda")
    cache = rq.KvCache(*((torch.randn((300, 2, 64, 128), generator=gen, device="cuda").half()) for _ in range(2)))
    q = torch.randn((fresh, 8, 128), generator=gen, device="cuda")

    def call():
        return ctx.attention(q, cache, torch.arange(300, **i32)[None], torch.tensor([0, fresh], **i32), torch.tensor([19_000], **i32), max_fresh=fresh)

    want = call()
    ctx.check()
    ctx.set_wait_limit(2_000_000)
    ctx.wait_selftest()
    with pytest.raises(rq.RqError, match="self-test"):
        ctx.check()
    ctx.set_wait_limit(2_000_000_000)
    for _ in range(3):
        assert torch.equal(call(), want)
    ctx.check()
    ctx.close()
