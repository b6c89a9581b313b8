"""Waits of the tensor-core attention kernel end by themselves, whichever warp gives up (no GPU: read from the sources)."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "recipe_dev_b200" / "csrc"


def source():
    return "\n".join(line.split("//")[0] for line in (CSRC / "rq_attention_tc.cu").read_text().splitlines())


def test_no_role_waits_without_a_limit():
    """A barrier of the hardware knows no limit: a warp that gave up and left would be missing at it for good. The two that all warps meet at are the ones before
    the roles part, and the one behind all of them, which every way out of a role leads to."""
    kernel = source().split("rq_attention_tc_kernel(")[1].split("\ntemplate")[0]
    roles = kernel[kernel.index("auto next_item") : kernel.rindex("__syncthreads();")]
    assert not re.search(r"bar\.sync|barrier\.sync|__syncthreads|named_sync|__nanosleep|mbar_try_wait|\bmbar_wait\(", roles)
    assert "bar.sync" not in source()
    assert re.findall(r"[^\n;{}]*\breturn;", roles) == ["                    if (!active) return;"]  # (of the function that writes a row)
    assert all("p.wait_ns" in w for w in re.findall(r"mbar_wait_warp\([^;]*;", kernel))


def test_the_work_area_has_a_count_for_every_warp_of_rows():
    shared = (CSRC / "rq_attention.cuh").read_text()
    ctas = int(re.search(r"kTensorCtas = (\d+)", shared)[1])
    rows = int(eval(re.search(r"kRowCtas = ([\d* ]+)", shared)[1]))
    counts = re.search(r"constexpr size_t kCounts = (.*);", shared)[1]
    assert counts == "kTensorCtas * 2 * 4 > kRowCtas ? kTensorCtas * 2 * 4 : kRowCtas" and rows <= ctas * 2 * 4
    host = (CSRC / "rq_attention.cu").read_text()
    assert host.count("kCounts * sizeof(uint32_t)") == 2 and "kRowCtas * sizeof" not in host
