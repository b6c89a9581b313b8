"""A kernel's opt-in to large shared memory or to large clusters is an attribute on one device: it is set at every call, or remembered by device (no GPU: read
from the sources)."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "recipe_dev_b200" / "csrc"
NAMES = ("cudaFuncSetAttribute(", "cudaOccupancyMaxActiveBlocksPerMultiprocessor(")


def functions(text):
    """The bodies at file or namespace level, comments taken out."""
    code = "\n".join(line.split("//")[0] for line in text.splitlines())
    for head in re.finditer(r"^(?!namespace|struct|extern|typedef|#)[^\n;{}]*\)\s*\{\n", code, re.M):
        end = code.index("\n}", head.end())
        yield code[head.start() : end]


def test_nothing_set_on_one_device_is_taken_for_set_on_another():
    found = 0
    for path in [*CSRC.glob("*.cu"), *CSRC.glob("*.cuh")]:
        for body in functions(path.read_text()):
            if not any(n in body for n in NAMES):
                continue
            found += 1
            kept = re.findall(r"\bstatic (?!const)[\w:]+ (\w+)(\[\w+\])?(?:\[\w+\])*(?= =|;)", body)
            assert all(size == "[64]" for _, size in kept), (path.name, kept)
            for name, _ in kept:
                places = re.findall(rf"\b{name}\[([^\]]+)\]", body)
                assert places and set(places) - {"64"} <= {"dev", "ctx->device"}, (path.name, name, places)
    assert found >= 10
