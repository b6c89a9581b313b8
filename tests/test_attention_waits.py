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
    assert host.count("kCounts * sizeof(uint32_t)") == 3 and "kRowCtas * sizeof" not in host


def test_a_role_that_gave_up_hands_nothing_on():
    """Armed or arrived at once more, a barrier whose copies are in flight would count what it does not expect; a tile on its way is not mended."""
    kernel = source().split("rq_attention_tc_kernel(")[1]
    issuing, rest = kernel.split("if (warp == kIssuer) {\n        \n")[1].split("} else if (warp == kFetcher)")
    mending, loading = rest.split("} else if (warp == kMender)")[1].split("} else if (warp == kLoader)")
    # the issuing warp: products and commits
    for body in re.findall(r"if \(elect_one\(\)([^)]*)\)", issuing):
        assert body == " && !dead"
    assert issuing.count("elect_one()") == issuing.count("elect_one() && !dead") == 3
    last = issuing[issuing.index("dead = false;") :]
    assert last.index("release(&sh.ended);") < last.index("arrived(&sh.ended, 0)") and issuing.count("sh.ended") == 2
    # the mending warp
    waited = mending.index("&sh.landed[slot]")
    assert waited < mending.index("if (dead) break;") < mending.index("uint4* v") < mending.index("mbar_arrive(&sh.full[slot])")
    # the loading warp: neither slots nor items
    tiles = loading[loading.index("&sh.empty[slot]") :]
    assert tiles.index("if (dead) break;") < tiles.index("mbar_expect_tx(") < tiles.index("tma_load_4d(")
    assert "while (following.take && !dead)" in loading
    assert re.search(r"if \(lane == 0 && !dead\) \{\s*sh\.items\[item_at\.slot\] = i;\s*mbar_arrive\(&sh\.item_full", loading)


def test_every_copy_has_landed_before_the_cta_ends():
    """The loading warp waits for each slot's last copies at the barriers that they are counted by, whether it gave up or another role did."""
    loading = source().split("} else if (warp == kLoader)")[1].split("tcgen05.dealloc")[0]
    copies, last = loading.split("for (int n = 0; n < 2 * STAGES; ++n)")
    assert copies.count("tma_load_4d(") == 1 and re.search(r"bar = &sh\.landed\[slot\];\s*landings \^= 1u << slot;", copies)
    assert "const int slot = n >> 1;" in last and last.count("late);") == 2 and last.count("bool late = false;") == 1
    assert "mbar_wait_warp(&sh.landed[slot], (landings >> slot & 1) ^ 1," in last and "mbar_wait_warp(&sh.full[slot], slot < at.slot ? at.phase : at.phase ^ 1," in last
    assert not re.search(r"\bif \(dead\)", last) and last.index("mbar_wait_warp(") < last.index("__syncthreads();")


def test_the_parities_that_the_last_waits_look_at():
    """A wait of parity q is over when the phase before the one that runs has that parity: it must be the phase of the slot's last fill, and of its last landing, for
    every length and mixture."""
    import random

    rng = random.Random(2)
    for stages in (3, 4, 5, 8):
        for fills in range(5 * stages):
            full, landed = [0] * stages, [0] * stages  # completed phases: by the copies themselves, or by the mending warp behind them
            landings = at = phase = 0
            for edge in (rng.random() < 0.4 for _ in range(fills)):
                full[at] += 1
                landed[at] += edge
                landings ^= edge << at
                at, phase = (at + 1, phase) if at + 1 < stages else (0, phase ^ 1)
            for slot in range(stages):  # (none: the phase before the first one has parity 1)
                assert (landings >> slot & 1) ^ 1 == (landed[slot] - 1) & 1
                assert (phase if slot < at else phase ^ 1) == (full[slot] - 1) & 1


def test_a_check_that_reports_a_wait_clears_what_was_counted():
    """A CTA that gave up leaves the counts of parts short: the next call would join rows before all of their parts are there."""
    api = (CSRC / "rq_api.cu").read_text().split('extern "C" int rq_check(')[1].split("\n}")[0]
    reported = api.split("if (flag) {")[1]
    assert reported.index("rq_attention_forget(ctx)") < reported.index("cudaMemset(ctx->error_flag, 0") < reported.index("cudaDeviceSynchronize()") < reported.index("RQ_ERR_WAIT")
    forget = (CSRC / "rq_attention.cu").read_text().split("int rq_attention_forget(rq_ctx* ctx) {")[1].split("\n}")[0]
    assert "if (ctx->attn_scratch) RQ_CUDA(cudaMemset(ctx->attn_scratch + kPartialBytes, 0, kCounts * sizeof(uint32_t)));" in forget
