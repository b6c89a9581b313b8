"""A host that has its weights and activations in numpy arrays needs no torch: neither the module nor a context imports it (no GPU needed; with one, a product runs)."""
import subprocess
import sys
from pathlib import Path

PROGRAM = """
import sys
sys.modules["torch"] = None  # an import of it raises
import numpy as np
import recipe_dev_b200 as rq
try:
    ctx = rq.Context(0)
except rq.RqError as e:
    print("no device:", e)
    sys.exit(0)
blocks = np.zeros(4 * 34 * 8, dtype=np.uint8)
y = ctx.matvec_host(ctx.weight_from_host(rq.Q8_0, blocks, 4, 256), np.ones((1, 256), dtype=np.float32))
assert (y == 0).all()
ctx.check()
ctx.close()
"""


def test_a_context_without_torch():
    run = subprocess.run([sys.executable, "-c", PROGRAM], capture_output=True, text=True, timeout=120, cwd=Path(__file__).resolve().parent.parent)
    assert run.returncode == 0, run.stderr[-2000:]
